// The product of E4M3 operands with one fp32 scale for each block of 128 (sm_100a), dense and for rows sorted by expert:
//
//   C[m, n] = sum over kb of sa[m, kb] * sb[n / 128, kb] * dot(A[m, 128 kb ..], B[n, 128 kb ..])   (+ bias[n])
//
// A [rows, K] and B [N, K] (or [experts, N, K]) are E4M3 bytes, K contiguous; sa is fp32 with one value for each row and
// 128 columns, sb one for each 128 x 128 tile: the checkpoint format that
// amct_pytorch/experimental/quantization/DeepSeekV3.2/deploy.py:48-90 dequantizes.  The scales may be any fp32
// numbers, which the MMA cannot apply (its block scales are powers of two; scales that happen to be powers of two are folded
// like the others): the tensor core sums 128 products into tensor memory, and the epilogue warps fold that partial sum, times
// fl(sa * sb), into fp32 registers.  A product sa * sb outside the normal range of fp32 loses bits or overflows.  Against 64
// bits the fp32 results are within 2^-21 of the sum of magnitudes for every kind of codes tried (normal, uniform bytes, one
// large code among small ones; K from 128 to 8192), which is what an fp32 matrix product of the same numbers has; the
// hardware documents no bound for its 128-long sums.  A tensor-memory
// buffer holds ONE K block; there are several, so that the MMAs of the next blocks run while a block is folded in.
//
// Two kernels, both with a TMA producer warp, one MMA-issuing thread and epilogue warps:
//   wide    128 rows of A x 256 columns, persistent.  A lane owns a row, so sa * sb is one number per K block and the fold
//           is one FMA per element.  Bound by the operands' way into the SM, close to it by the folding's hand-over.
//   narrow  for few rows (a decode batch): the weight is the 128-row MMA operand, 16 to 128 tokens are its columns.  Bound
//           by the weight's bytes; K is split over a thread-block cluster whose CTAs add their partial sums through
//           distributed shared memory in rank order, so a small weight still occupies every SM and results repeat.
//           1 x 14336 x 4096: 15 us, of which 9 are the weight's 59 MB at the copy rate, 3 the way to the first operands
//           and 2 the join; 128 rows on 32 experts of 4096 x 7168 (940 MB): 131 to 144 us, the copy rate.
// Grouped: offsets [experts + 1] on the device say which rows belong to which expert.  Every CTA builds the table of
// row tiles from them; a tile may read rows of the next expert (it never stores them).  Offsets that are out of
// range or not ascending are clamped to a running maximum within [0, rows]: no access depends on their values.
//
// K need not be a multiple of 128: the tensor maps end at K and the rest of the last block reads as zero.
#include <cuda.h>

#include "common.cuh"
#include "tc05.cuh"

namespace amct {
namespace f8g {

constexpr int kBlock = 128;                     // rows of an MMA tile, and bytes of K per pipeline stage
constexpr int kMaxExperts = 1024;
// A wait that ran out leaves NaN in every output that it leaves unknown, besides its bit in the status word: a failure shows
// without a host read, and without a status word.
__device__ __forceinline__ float unknown() { return __int_as_float(0x7fffffff); }

struct Params {
  int64_t m, n, k;
  const float* sa;
  int64_t sa_row, sa_k;        // strides in elements
  const float* sb;
  int64_t sb_expert, sb_row, sb_k;
  const void* bias;
  int bias_kind;               // AMCT_BIAS_NONE / F32 / F16 / BF16
  void* out;
  int out_kind;                // AMCT_GEMM_OUT_F32 / F16 / BF16
  int64_t ld_out;
  const int* offsets;          // [experts + 1], or null: one group of m rows
  int experts;
  int group_m;                 // wide kernel, dense: row tiles per rasterisation group
  int* status;
};

// ---------------------------------------------------------------------------------------------- row tiles of the groups
struct GroupTable {
  int bound[kMaxExperts + 1];  // first row of every group, made ascending
  int first[kMaxExperts + 1];  // first row tile of every group
};

// Whole block; THREADS a multiple of 32.
template <int THREADS, int TILE>
__device__ __forceinline__ void build_groups(const Params& p, GroupTable& g) {
  const int n = p.experts + 1;
  const int rows = (int)p.m;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const int v = __ldg(p.offsets + i);
    g.bound[i] = v < 0 ? 0 : v > rows ? rows : v;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, per = (n + 31) / 32;
    const int lo = lane * per < n ? lane * per : n, hi = lo + per < n ? lo + per : n;
    int top = 0;
    for (int i = lo; i < hi; ++i) top = max(top, g.bound[i]);
    int incl = top;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl = max(incl, v);
    }
    int run = __shfl_up_sync(0xffffffffu, incl, 1);
    if (lane == 0) run = 0;
    for (int i = lo; i < hi; ++i) {
      run = max(run, g.bound[i]);
      g.bound[i] = run;
    }
    __syncwarp();
    int sum = 0;
    for (int i = lo; i < hi; ++i) sum += i < p.experts ? (g.bound[i + 1] - g.bound[i] + TILE - 1) / TILE : 0;
    incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    int at = incl - sum;
    for (int i = lo; i < hi; ++i) {
      g.first[i] = at;
      at += i < p.experts ? (g.bound[i + 1] - g.bound[i] + TILE - 1) / TILE : 0;
    }
  }
  __syncthreads();
}

struct Tile {
  int row0, row_end;           // rows [row0, min(row0 + tile, row_end)) are this tile's
  int tn;                      // column tile
  int expert;
};

// Tile numbers are 32-bit (the launcher sees to it): a 64-bit division per tile would cost every role its registers.
// Grouped: all tiles of a group lie together, row tiles fastest, so that CTAs running at one time share its weight.
template <int TILE>
__device__ __forceinline__ Tile group_tile(const Params& p, const GroupTable& g, uint32_t tile, uint32_t tiles_n) {
  const int want = (int)(tile / tiles_n);
  int lo = 0, hi = p.experts;                    // first[lo] <= want < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (g.first[mid] <= want) lo = mid; else hi = mid;
  }
  Tile t;
  t.expert = lo;
  const uint32_t rel = tile - (uint32_t)g.first[lo] * tiles_n;
  const uint32_t mt = (uint32_t)(g.first[lo + 1] - g.first[lo]);
  t.tn = (int)(rel / mt);
  t.row0 = g.bound[lo] + (int)(rel - (uint32_t)t.tn * mt) * TILE;
  t.row_end = g.bound[lo + 1];
  return t;
}

template <int TILE>
__device__ __forceinline__ Tile dense_tile(const Params& p, uint32_t tile, uint32_t tiles_m, uint32_t tiles_n) {
  const uint32_t per_group = (uint32_t)p.group_m * tiles_n;
  const uint32_t g = tile / per_group, r = tile - g * per_group;
  const uint32_t m0 = g * (uint32_t)p.group_m;
  const uint32_t gm = tiles_m - m0 < (uint32_t)p.group_m ? tiles_m - m0 : (uint32_t)p.group_m;
  Tile t;
  t.tn = (int)(r / gm);
  t.row0 = (int)(m0 + (r - (uint32_t)t.tn * gm)) * TILE;
  t.row_end = (int)p.m;
  t.expert = 0;
  return t;
}

// a bounded wait of a whole warp: all of its lanes go on, or none
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, tc05::mbar_wait(bar, parity, abort_flag));
}

__device__ __forceinline__ float bias_at(const Params& p, int64_t n) {
  switch (p.bias_kind) {
    case AMCT_BIAS_F32: return reinterpret_cast<const float*>(p.bias)[n];
    case AMCT_BIAS_F16: return __half2float(reinterpret_cast<const __half*>(p.bias)[n]);
    case AMCT_BIAS_BF16: return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.bias)[n]);
  }
  return -0.f;                                   // x + (-0) is x for every x
}

// ---------------------------------------------------------------------------------------------- wide kernel
// Three warpgroups: TMA and MMA warps in the first (two of its warps idle), eight folding warps in the others.  The launch
// gives every thread 168 registers; the first group hands back all but 40, the folding groups take 232 (40 + 2 x 232 =
// 3 x 168): 128 sums and two 16-column loads without a spill.
//
// What bounds it: 48 KB of operands for each K block, 64 bytes a cycle into an SM: 769 cycles (measured with the folding
// left out; the block's MMAs alone take 520).  With the folding it is 880: a buffer's round -- MMAs until seen done 740,
// loads 250, hand-over 250, for two buffers -- is close behind.  8192 x 8192 x 8192 back to back: 556 us = 1.98 PFLOP/s at
// 1.43 GHz (the board's power limit); 8192 x 7168 x 8192: 435 us = 2.2 PFLOP/s for ten in a row from cool, 507 us = 1.9 in a
// sequence of calls.
// Measured and left out: CTA pairs (32 KB for each block, but the hand-over crosses CTAs: 1 % faster at the largest size,
// 15 to 80 % slower at 4096 x 7168 x 2048, 777 x 5120 x 4096 and for experts with 500 rows); sixteen folding warps (20 %
// slower); paired FMAs (fma.rn.f32x2, 1.6 times the time); scales staged by a warp of their own (10 % slower); unrolling
// the K loop by two (20 % slower: the folding code outgrows the instruction cache); one lane polling for its warp (25 %).
constexpr int kWideN = 256, kWideStages = 4, kWideEpiWarps = 8, kWideThreads = 128 + 32 * kWideEpiWarps;
constexpr int kWideRegsFirst = 40, kWideRegsFold = 232;
constexpr int kWideA = kBlock * kBlock, kWideB = kWideN * kBlock, kWideStageBytes = kWideA + kWideB;

constexpr int kTurnBytes = 32 * 64;      // per folding warp: 64 bytes of 32 rows

struct __align__(1024) WideSmem {
  uint8_t tiles[kWideStages][kWideStageBytes];
  uint8_t turn[kWideEpiWarps][kTurnBytes];
  GroupTable groups;
  uint64_t full[kWideStages], empty[kWideStages], tmem_full[2], tmem_empty[2];
  uint32_t tmem_base;
  volatile int abort_flag;
};


// A folding warp's 32 rows x 128 columns, 64 bytes of every row at a time.  A lane holds a row, so the values turn around in
// shared memory first and leave with neighbouring lanes on neighbouring outputs, where a lane's own row would touch 32 lines
// with 16 bytes each:
//   rows at multiples of 16 bytes: 16 bytes to a lane, 8 rows for each instruction;
//   others (an odd N), and the last columns: a word to a lane, 2 rows for each instruction.  16-bit rows that begin in the
//   middle of a word are shifted by one output on their way into shared memory; their first and last output go alone.
// What counts is instructions: single outputs, 32 to an instruction, took three times as long for 4096 x 16001 x 128 as for
// 4096 x 16000 x 128 (140 us, 46; as it is 70, and 777 x 5001 x 4000 21.8 us, 20.8 with 5008 columns).
template <bool BIAS>
__device__ __forceinline__ void store_rows(const Params& p, int warp_row0, int row_end, int lane, int64_t n0, float (&acc)[128], uint8_t* turn) {
  const int esize = p.out_kind == AMCT_GEMM_OUT_F32 ? 4 : 2;
  const int rows = min(row_end - warp_row0, 32), bytes = (int)(p.n - n0 < 128 ? p.n - n0 : 128) * esize;      // what exists of them
  const int64_t ld = p.ld_out * esize;
  uint8_t* out = reinterpret_cast<uint8_t*>(p.out) + warp_row0 * ld + n0 * esize;
  const bool vectors = ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)ld) & 15) == 0;
  // rows in steps of two begin alike: `half` is the first or second half of the warp
  const int half = lane >> 4, odd = (int)((reinterpret_cast<uintptr_t>(out) + lane * ld) >> 1 & 1);
  const int odd_row = (int)((reinterpret_cast<uintptr_t>(out) + half * ld) >> 1 & 1);
  const uint32_t shift = odd ? 0x5432 : 0x7654;
  uint32_t last = 0;                             // word in front of the next
#pragma unroll
  for (int c0 = 0; c0 < 128; c0 += 32) {
    if (n0 + c0 > p.n) break;                    // at n0 + c0 == p.n a shifted row still has its last output to come
    float y[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) y[j] = acc[c0 + j];
    if constexpr (BIAS) {                        // one load for each lane, handed around
      const float b = n0 + c0 + lane < p.n ? bias_at(p, n0 + c0 + lane) : 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j) y[j] = __fadd_rn(y[j], __shfl_sync(0xffffffffu, b, j));
    }
    uint32_t h[32];                              // the 32 outputs as they are stored: 16 or 32 words
    if (esize == 2) {
      uint32_t packed[16];
      epi_pack16(y, p.out_kind == AMCT_GEMM_OUT_BF16, packed);
      if (vectors) {
#pragma unroll
        for (int j = 0; j < 16; ++j) h[j] = packed[j];
      } else {
        if (c0 == 0 && odd && lane < rows) *reinterpret_cast<uint16_t*>(out + lane * ld) = (uint16_t)packed[0];
#pragma unroll
        for (int j = 0; j < 16; ++j) h[j] = __byte_perm(j ? packed[j ? j - 1 : 0] : last, packed[j], shift);
        last = packed[15];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) h[j] = __float_as_uint(y[j]);
    }
#pragma unroll
    for (int part = 0; part < 2; ++part) {       // 64 bytes of every row; one part of 16-bit outputs, two of fp32
      if (part * 16 * 4 >= 32 * esize) break;
      const int at = c0 * esize + part * 64;
#pragma unroll
      for (int q = 0; q < 4; ++q)                // chunk q of row r lies at chunk q ^ (r / 2 % 4): neither side conflicts
        *reinterpret_cast<uint4*>(turn + lane * 64 + ((q ^ (lane >> 1)) & 3) * 16) =
            make_uint4(h[part * 16 + 4 * q], h[part * 16 + 4 * q + 1], h[part * 16 + 4 * q + 2], h[part * 16 + 4 * q + 3]);
      __syncwarp();
      if (vectors && at + 64 <= bytes) {
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int r = it * 8 + (lane >> 2), q = lane & 3;
          if (r < rows) *reinterpret_cast<uint4*>(out + r * ld + at + q * 16) = *reinterpret_cast<const uint4*>(turn + r * 64 + ((q ^ (r >> 1)) & 3) * 16);
        }
      } else {
        const int word = lane & 15, mine = at + word * 4 - 2 * odd_row;
        const uint8_t* from = turn + half * 64 + (word & 3) * 4;
        uint8_t* to = out + half * ld + mine;
        const int whole = mine >= 0 && mine + 4 <= bytes ? rows - half : 0;     // rows whose word is this lane's to store
        const int part_of = mine >= 0 && mine + 2 == bytes ? rows - half : 0;   // ... whose last output is in it, alone
#pragma unroll
        for (int it = 0; it < 16; ++it) {
          const uint32_t v = *reinterpret_cast<const uint32_t*>(from + it * 128 + (((word >> 2) ^ it) & 3) * 16);
          if (it * 2 < whole) *reinterpret_cast<uint32_t*>(to) = v;
          to += 2 * ld;
        }
        if (bytes < 128 * esize) {
          to = out + half * ld + mine;
#pragma unroll 1
          for (int it = 0; it * 2 < part_of; ++it, to += 2 * ld)
            *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from + it * 128 + (((word >> 2) ^ it) & 3) * 16);
        }
      }
      __syncwarp();
    }
  }
  if (odd && !vectors && esize == 2 && bytes == 256 && lane < rows) *reinterpret_cast<uint16_t*>(out + lane * ld + 254) = (uint16_t)(last >> 16);
}

// BIAS is a parameter because its code, never run, still costs the folding loop 2 %.
template <bool GROUPED, bool BIAS>
__global__ void __launch_bounds__(kWideThreads, 1)
gemm_fp8_wide_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, Params p) {
  extern __shared__ uint8_t smem_raw[];
  WideSmem& s = *reinterpret_cast<WideSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_kb = (int)((p.k + kBlock - 1) / kBlock);
  const uint32_t tiles_n = (uint32_t)((p.n + kWideN - 1) / kWideN);
  const uint32_t tiles_m = (uint32_t)((p.m + kBlock - 1) / kBlock);

  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    for (int i = 0; i < kWideStages; ++i) { tc05::mbar_init(tc05::smem_u32(&s.full[i]), 1); tc05::mbar_init(tc05::smem_u32(&s.empty[i]), 1); }
    for (int i = 0; i < 2; ++i) { tc05::mbar_init(tc05::smem_u32(&s.tmem_full[i]), 1); tc05::mbar_init(tc05::smem_u32(&s.tmem_empty[i]), kWideEpiWarps); }
    tc05::fence_barrier_init();
    tc05::prefetch_tmap(&tma_a);
    tc05::prefetch_tmap(&tma_b);
  }
  if (warp == 1) {
    tc05::tmem_alloc(tc05::smem_u32(&s.tmem_base), 512);
    tc05::tmem_relinquish();
  }
  if (GROUPED) build_groups<kWideThreads, kBlock>(p, s.groups);
  tc05::fence_before_sync();
  __syncthreads();
  tc05::fence_after_sync();
  const uint32_t tmem_base = s.tmem_base;
  volatile int* abort_flag = &s.abort_flag;
  const uint32_t num_tiles = (GROUPED ? (uint32_t)s.groups.first[p.experts] : tiles_m) * tiles_n;

  if (warp < 4) {
    tc05::regs_dec<kWideRegsFirst>();
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer
      if (tc05::elect_one()) {
        uint32_t stage = 0, phase = 0;
        bool alive = true;
        for (uint32_t tile = blockIdx.x; tile < num_tiles && alive; tile += gridDim.x) {
          const Tile t = GROUPED ? group_tile<kBlock>(p, s.groups, tile, tiles_n) : dense_tile<kBlock>(p, tile, tiles_m, tiles_n);
          const int row_b = t.expert * (int)p.n + t.tn * kWideN;
          for (int kb = 0; kb < num_kb; ++kb) {
            if (!tc05::mbar_wait(tc05::smem_u32(&s.empty[stage]), phase ^ 1, abort_flag)) { alive = false; break; }
            const uint32_t bar = tc05::smem_u32(&s.full[stage]);
            tc05::mbar_expect_tx(bar, kWideStageBytes);
            const uint32_t dst = tc05::smem_u32(&s.tiles[stage][0]);
            tc05::tma_load_2d(dst, &tma_a, bar, kb * kBlock, t.row0);
            tc05::tma_load_2d(dst + kWideA, &tma_b, bar, kb * kBlock, row_b);
            if (++stage == kWideStages) { stage = 0; phase ^= 1; }
          }
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer: one tensor-memory buffer per K block
      if (tc05::elect_one()) {
        constexpr uint32_t idesc = tc05::make_idesc(1, 0, 0, kBlock, kWideN);
        uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
        bool alive = true;
        for (uint32_t tile = blockIdx.x; tile < num_tiles && alive; tile += gridDim.x) {
          for (int kb = 0; kb < num_kb; ++kb) {
            if (!tc05::mbar_wait(tc05::smem_u32(&s.full[stage]), phase, abort_flag)) { alive = false; break; }
            const uint32_t a0 = tc05::smem_u32(&s.tiles[stage][0]);
            const uint64_t a_desc = tc05::smem_desc_sw128(a0), b_desc = tc05::smem_desc_sw128(a0 + kWideA);
            if (!tc05::mbar_wait(tc05::smem_u32(&s.tmem_empty[buf]), buf_phase ^ 1, abort_flag)) { alive = false; break; }
            tc05::fence_after_sync();
#pragma unroll
            for (int ks = 0; ks < kBlock / 32; ++ks)         // 32 bytes along K: 2 in the descriptor's units
              tc05::umma_f8(tmem_base + buf * kWideN, a_desc + 2 * ks, b_desc + 2 * ks, idesc, ks > 0);
            tc05::umma_commit(tc05::smem_u32(&s.tmem_full[buf]));
            tc05::umma_commit(tc05::smem_u32(&s.empty[stage]));
            if (++stage == kWideStages) { stage = 0; phase ^= 1; }
            if (++buf == 2) { buf = 0; buf_phase ^= 1; }
          }
        }
      }
    }
  } else {
    tc05::regs_inc<kWideRegsFold>();
    // ------------------------------------------------------------ fold and store: 32 rows x 128 columns per warp
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t full0 = tc05::smem_u32(&s.tmem_full[0]), empty0 = tc05::smem_u32(&s.tmem_empty[0]);
    const uint32_t t_warp = tmem_base + ((uint32_t)(quarter * 32) << 16) + half * 128;
    uint32_t buf = 0, buf_phase = 0;
    bool alive = true;
    for (uint32_t tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
      const Tile t = GROUPED ? group_tile<kBlock>(p, s.groups, tile, tiles_n) : dense_tile<kBlock>(p, tile, tiles_m, tiles_n);
      const int row = t.row0 + quarter * 32 + lane;
      const int64_t n0 = (int64_t)t.tn * kWideN + half * 128;
      const bool row_in = row < t.row_end, cols_in = n0 < p.n;
      const float* sa = p.sa + (int64_t)(row_in ? row : t.row0) * p.sa_row;
      const float* sb = p.sb + (int64_t)t.expert * p.sb_expert + (cols_in ? n0 / kBlock : 0) * p.sb_row;
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.f;
      float next_a = __ldg(sa), b_32 = 0.f;      // b_32: lane l holds B's scale of block kb / 32 * 32 + l
#pragma unroll 1
      for (int kb = 0; kb < num_kb && alive; ++kb) {
        if ((kb & 31) == 0) b_32 = kb + lane < num_kb ? __ldg(sb + (kb + lane) * p.sb_k) : 0.f;
        const float f = __fmul_rn(next_a, __shfl_sync(0xffffffffu, b_32, kb & 31));
        sa += p.sa_k;
        if (kb + 1 < num_kb) next_a = __ldg(sa); // on its way while this block is folded
        if (!warp_wait(full0 + buf * 8, buf_phase, abort_flag)) { alive = false; break; }
        tc05::fence_after_sync();
        const uint32_t t_row = t_warp + buf * kWideN;
        uint32_t r[2][16];
        tc05::tmem_ld_32x16(t_row, r[0]);
#pragma unroll
        for (int c = 0; c < 7; ++c) {
          tc05::tmem_ld_wait(r[c & 1]);
          tc05::tmem_ld_32x16(t_row + (c + 1) * 16, r[(c + 1) & 1]);
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[c * 16 + j] = __fmaf_rn(__uint_as_float(r[c & 1][j]), f, acc[c * 16 + j]);
        }
        tc05::tmem_ld_wait(r[1]);
        tc05::fence_before_sync();               // everything read: the buffer goes back before the last folds
        __syncwarp();
        if (lane == 0) tc05::mbar_arrive(empty0 + buf * 8);
        buf_phase ^= buf;
        buf ^= 1;
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[112 + j] = __fmaf_rn(__uint_as_float(r[1][j]), f, acc[112 + j]);
      }
      if (!alive) {                              // a wait ran out: nothing of this tile or a later one is known
#pragma unroll
        for (int j = 0; j < 128; ++j) acc[j] = unknown();
      }
      if (cols_in) store_rows<BIAS>(p, t.row0 + quarter * 32, t.row_end, lane, n0, acc, s.turn[warp - 4]);
      __syncwarp();
    }
  }

  __syncthreads();
  if (*abort_flag) {
    if (warp >= 4) {                             // the warps that have registers to spare
      if (threadIdx.x == kWideThreads - 1 && p.status) atomicOr(p.status, 2);
      tc05::let_land();
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc05::fence_after_sync();
    tc05::tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------------------------- narrow kernel
constexpr int kNarrowBufs = 4, kMaxSplits = 8;

// Folding warps: four (32 weight rows each), or eight that also halve the columns, so that a lane holds at most 64 sums.
// Up to 64 tokens two CTAs share an SM (about 110 KB of shared memory each); 128 tokens take one alone.
template <int NT> constexpr int narrow_ctas() { return NT <= 64 ? 2 : 1; }
template <int NT> constexpr int narrow_stages() { return NT <= 32 ? 5 : NT <= 64 ? 4 : 6; }
template <int NT> constexpr int narrow_folders() { return NT <= 32 ? 4 : 8; }
template <int NT> constexpr int narrow_cols() { return NT * 4 / narrow_folders<NT>(); }
template <int NT> constexpr int narrow_threads() { return 64 + 32 * narrow_folders<NT>(); }

template <int NT>
struct __align__(1024) NarrowSmem {
  static constexpr int kStageBytes = (kBlock + NT) * kBlock;
  uint8_t tiles[narrow_stages<NT>()][kStageBytes];    // the K loop's ring, afterwards this CTA's partial sums [NT][128]
  float factor[narrow_folders<NT>()][2][narrow_cols<NT>()];      // sa * sb of a K block
  GroupTable groups;
  uint64_t full[narrow_stages<NT>()], empty[narrow_stages<NT>()], tmem_full[kNarrowBufs], tmem_empty[kNarrowBufs];
  uint32_t tmem_base;
  volatile int abort_flag;
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ int ld_cluster1(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

__device__ __forceinline__ void store_one(const Params& p, int64_t row, int64_t n, float v) {
  const int64_t off = row * p.ld_out + n;
  switch (p.out_kind) {
    case AMCT_GEMM_OUT_F32: reinterpret_cast<float*>(p.out)[off] = v; break;
    case AMCT_GEMM_OUT_F16: reinterpret_cast<__half*>(p.out)[off] = __float2half_rn(v); break;
    default: reinterpret_cast<__nv_bfloat16*>(p.out)[off] = __float2bfloat16_rn(v);
  }
}

// four consecutive outputs of a row
__device__ __forceinline__ void store_four(const Params& p, int64_t row, int64_t n, float4 v) {
  const int64_t off = row * p.ld_out + n;
  if (p.out_kind != AMCT_GEMM_OUT_F32 && n + 3 < p.n && ((reinterpret_cast<uintptr_t>(p.out) + 2 * off) & 7) == 0) {
    uint2 h;
    if (p.out_kind == AMCT_GEMM_OUT_BF16) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
      h = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
      const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
      h = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + off) = h;
    return;
  }
  const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < p.n) store_one(p, row, n + i, f[i]);
}

// Grid: splits CTAs (one cluster) for each tile.  CTA `rank` of a cluster takes the K blocks
// [rank * num_kb / splits, (rank + 1) * num_kb / splits).
template <int NT, bool GROUPED>
__global__ void __launch_bounds__(narrow_threads<NT>(), narrow_ctas<NT>())
gemm_fp8_narrow_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_x, Params p, int splits) {
  constexpr int kStages = narrow_stages<NT>();
  constexpr uint32_t kTmemCols = NT * kNarrowBufs < 32 ? 32 : NT * kNarrowBufs;
  extern __shared__ uint8_t smem_raw[];
  NarrowSmem<NT>& s = *reinterpret_cast<NarrowSmem<NT>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = splits > 1 ? tc05::cluster_ctarank() : 0;
  const int num_kb_all = (int)((p.k + kBlock - 1) / kBlock);
  const int kb_lo = (int)((int64_t)num_kb_all * rank / splits), kb_hi = (int)((int64_t)num_kb_all * (rank + 1) / splits);
  const uint32_t tiles_n = (uint32_t)((p.n + kBlock - 1) / kBlock);
  const uint32_t tile = blockIdx.x / (uint32_t)splits;

  Tile t;
  if (GROUPED) {
    build_groups<narrow_threads<NT>(), NT>(p, s.groups);
    if (tile >= (uint32_t)s.groups.first[p.experts] * tiles_n) return;      // the whole cluster leaves
    t = group_tile<NT>(p, s.groups, tile, tiles_n);
  } else {
    const uint32_t tiles_m = (uint32_t)((p.m + NT - 1) / NT);
    t.tn = (int)(tile / tiles_m);                // row tiles fastest: they share a slice of the weight
    t.row0 = (int)(tile - (uint32_t)t.tn * tiles_m) * NT;
    t.row_end = (int)p.m;
    t.expert = 0;
  }
  const int64_t n0 = (int64_t)t.tn * kBlock;

  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    for (int i = 0; i < kStages; ++i) { tc05::mbar_init(tc05::smem_u32(&s.full[i]), 1); tc05::mbar_init(tc05::smem_u32(&s.empty[i]), 1); }
    for (int i = 0; i < kNarrowBufs; ++i) { tc05::mbar_init(tc05::smem_u32(&s.tmem_full[i]), 1); tc05::mbar_init(tc05::smem_u32(&s.tmem_empty[i]), narrow_folders<NT>()); }
    tc05::fence_barrier_init();
    tc05::prefetch_tmap(&tma_w);
    tc05::prefetch_tmap(&tma_x);
  }
  if (warp == 1) {
    tc05::tmem_alloc(tc05::smem_u32(&s.tmem_base), kTmemCols);
    tc05::tmem_relinquish();
  }
  tc05::fence_before_sync();
  __syncthreads();
  tc05::fence_after_sync();
  const uint32_t tmem_base = s.tmem_base;
  volatile int* abort_flag = &s.abort_flag;
  if (warp == 0) {
    if (tc05::elect_one()) {
      uint32_t stage = 0, phase = 0;
      const int row_w = t.expert * (int)p.n + t.tn * kBlock;
      for (int kb = kb_lo; kb < kb_hi; ++kb) {
        if (!tc05::mbar_wait(tc05::smem_u32(&s.empty[stage]), phase ^ 1, abort_flag)) break;
        const uint32_t bar = tc05::smem_u32(&s.full[stage]);
        tc05::mbar_expect_tx(bar, NarrowSmem<NT>::kStageBytes);
        const uint32_t dst = tc05::smem_u32(&s.tiles[stage][0]);
        tc05::tma_load_2d(dst, &tma_w, bar, kb * kBlock, row_w);
        tc05::tma_load_2d(dst + kBlock * kBlock, &tma_x, bar, kb * kBlock, t.row0);
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (tc05::elect_one()) {
      constexpr uint32_t idesc = tc05::make_idesc(1, 0, 0, kBlock, NT);
      uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
      for (int kb = kb_lo; kb < kb_hi; ++kb) {
        if (!tc05::mbar_wait(tc05::smem_u32(&s.tmem_empty[buf]), buf_phase ^ 1, abort_flag)) break;
        if (!tc05::mbar_wait(tc05::smem_u32(&s.full[stage]), phase, abort_flag)) break;
        tc05::fence_after_sync();
        const uint32_t w0 = tc05::smem_u32(&s.tiles[stage][0]);
        const uint32_t x0 = w0 + kBlock * kBlock;
#pragma unroll
        for (int ks = 0; ks < kBlock / 32; ++ks)
          tc05::umma_f8(tmem_base + buf * NT, tc05::smem_desc_sw128(w0 + ks * 32), tc05::smem_desc_sw128(x0 + ks * 32), idesc, ks > 0);
        tc05::umma_commit(tc05::smem_u32(&s.empty[stage]));
        tc05::umma_commit(tc05::smem_u32(&s.tmem_full[buf]));
        if (++stage == kStages) { stage = 0; phase ^= 1; }
        if (++buf == kNarrowBufs) { buf = 0; buf_phase ^= 1; }
      }
    }
    __syncwarp();
  } else {
    constexpr int kCols = narrow_cols<NT>(), kPart = kCols < 32 ? kCols : 32, kPer = (kCols + 31) / 32;
    const int quarter = warp & 3, col0 = ((warp - 2) >> 2) * kCols;
    float(&factor)[2][kCols] = s.factor[warp - 2];
    const float* sb = p.sb + (int64_t)t.expert * p.sb_expert + (int64_t)t.tn * p.sb_row;
    const float* sa[kPer];                       // tokens whose scale this lane fetches
    float a_scale[kNarrowBufs][kPer], b_scale[kNarrowBufs];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = i * 32 + lane, row = t.row0 + col0 + c;
      sa[i] = p.sa + (int64_t)(c < kCols && row < t.row_end ? row : t.row0) * p.sa_row;
    }
    // scales as many blocks ahead as there are buffers: a load from L2 takes longer than a block
#pragma unroll
    for (int u = 0; u < kNarrowBufs; ++u) {
      const int64_t kb = kb_lo + u < kb_hi ? kb_lo + u : kb_lo;
      b_scale[u] = __ldg(sb + kb * p.sb_k);
#pragma unroll
      for (int i = 0; i < kPer; ++i) a_scale[u][i] = __ldg(sa[i] + kb * p.sa_k);
    }
    float acc[kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j) acc[j] = 0.f;
    uint32_t buf_phase = 0;
    bool alive = true;
    for (int base = kb_lo; base < kb_hi && alive; base += kNarrowBufs, buf_phase ^= 1) {
#pragma unroll
      for (int u = 0; u < kNarrowBufs; ++u) {    // u: buffer of the block
        const int kb = base + u;
        if (kb >= kb_hi) break;
        float(&f_now)[kCols] = factor[u & 1];
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (i * 32 + lane < kCols) f_now[i * 32 + lane] = __fmul_rn(a_scale[u][i], b_scale[u]);
        __syncwarp();                            // also: every lane has left the other side, which is written next
        if (kb + kNarrowBufs < kb_hi) {
          const int64_t later = kb + kNarrowBufs;
          b_scale[u] = __ldg(sb + later * p.sb_k);
#pragma unroll
          for (int i = 0; i < kPer; ++i) a_scale[u][i] = __ldg(sa[i] + later * p.sa_k);
        }
        if (!warp_wait(tc05::smem_u32(&s.tmem_full[u]), buf_phase, abort_flag)) { alive = false; break; }
        tc05::fence_after_sync();
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += kPart) {
          uint32_t r[kPart];
          const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16) + u * NT + col0 + c0;
          if constexpr (kPart == 16) tc05::tmem_ld_32x16(at, r);
          else tc05::tmem_ld_32x32(at, r);
          float4 f[kPart / 4];                   // on their way while the tensor memory answers
#pragma unroll
          for (int j = 0; j < kPart / 4; ++j) f[j] = *reinterpret_cast<const float4*>(&f_now[c0 + 4 * j]);
          tc05::tmem_ld_wait(r);
          if (c0 + kPart == kCols) {
            tc05::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc05::mbar_arrive(tc05::smem_u32(&s.tmem_empty[u]));
          }
#pragma unroll
          for (int j = 0; j < kPart / 4; ++j) {
            acc[c0 + 4 * j] = __fmaf_rn(__uint_as_float(r[4 * j]), f[j].x, acc[c0 + 4 * j]);
            acc[c0 + 4 * j + 1] = __fmaf_rn(__uint_as_float(r[4 * j + 1]), f[j].y, acc[c0 + 4 * j + 1]);
            acc[c0 + 4 * j + 2] = __fmaf_rn(__uint_as_float(r[4 * j + 2]), f[j].z, acc[c0 + 4 * j + 2]);
            acc[c0 + 4 * j + 3] = __fmaf_rn(__uint_as_float(r[4 * j + 3]), f[j].w, acc[c0 + 4 * j + 3]);
          }
        }
      }
    }
    // Every copy and every MMA of this CTA has completed (the last tensor-memory buffer was full): the ring is free.  The
    // sums turn around in it, so that a warp stores 128 consecutive outputs of a token.
    float* partial = reinterpret_cast<float*>(&s.tiles[0][0]);
#pragma unroll
    for (int j = 0; j < kCols; ++j) partial[(col0 + j) * kBlock + quarter * 32 + lane] = acc[j];
  }

  __syncthreads();
  if (splits > 1) {
    tc05::cluster_arrive();
    tc05::cluster_wait();
  }
  if (warp >= 2) {
    // Column j belongs to CTA j % splits, and there to one of its folding warps; a lane takes four consecutive outputs.  All
    // CTAs' partial sums are on their way before the first is added; they are added in rank order.  A CTA whose wait ran out
    // has only garbage to give: lane q looks at CTA q's flag, while the sums are on their way too.
    int failed = 0;
    if (splits == 1) failed = *abort_flag;
    else if (lane < splits) failed = ld_cluster1(tc05::map_to_cta(tc05::smem_u32(const_cast<const int*>(&s.abort_flag)), lane));
    const int64_t n = n0 + lane * 4;
    float b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = n + i < p.n ? bias_at(p, n + i) : 0.f;
    const uint32_t mine = tc05::smem_u32(&s.tiles[0][0]) + lane * 16;
    for (int j = (int)rank + (warp - 2) * splits; j < NT; j += narrow_folders<NT>() * splits) {
      if (t.row0 + j >= t.row_end) break;
      float4 sum;
      if (splits == 1) {
        sum = *reinterpret_cast<const float4*>(&s.tiles[0][0] + j * kBlock * 4 + lane * 16);
      } else {
        float4 part[kMaxSplits];
#pragma unroll
        for (int q = 0; q < kMaxSplits; ++q)
          if (q < splits) part[q] = ld_cluster4(tc05::map_to_cta(mine + j * kBlock * 4, q));
        sum = part[0];
#pragma unroll
        for (int q = 1; q < kMaxSplits; ++q) {
          if (q < splits) {
            sum.x = __fadd_rn(sum.x, part[q].x);
            sum.y = __fadd_rn(sum.y, part[q].y);
            sum.z = __fadd_rn(sum.z, part[q].z);
            sum.w = __fadd_rn(sum.w, part[q].w);
          }
        }
      }
      if (__any_sync(0xffffffffu, failed)) sum = make_float4(unknown(), unknown(), unknown(), unknown());
      store_four(p, t.row0 + j, n, make_float4(__fadd_rn(sum.x, b[0]), __fadd_rn(sum.y, b[1]), __fadd_rn(sum.z, b[2]), __fadd_rn(sum.w, b[3])));
    }
  }
  if (splits > 1) {
    __syncwarp();
    tc05::cluster_arrive();                      // nobody leaves while its partial sums are being read
    tc05::cluster_wait();
  }
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, 2);
    tc05::let_land();
    __syncthreads();
  }
  if (warp == 1) {
    tc05::fence_after_sync();
    tc05::tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------- host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// [rows, k] bytes -> tensor map with boxes of 128 bytes x box_rows rows, 128-byte swizzle
static int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return AMCT_ERR_CUDA;
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)kBlock, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? AMCT_OK : AMCT_ERR_CUDA;
}

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n;
}

template <bool GROUPED, bool BIAS>
static int launch_wide(const void* a, const void* b, int64_t ld_a, int64_t ld_b, int64_t rows_b, Params p, int sms, cudaStream_t st) {
  CUtensorMap ma, mb;
  int rc = make_map(&ma, a, p.m, p.k, ld_a, kBlock);
  if (rc != AMCT_OK) return rc;
  rc = make_map(&mb, b, rows_b, p.k, ld_b, kWideN);
  if (rc != AMCT_OK) return rc;
  const size_t smem = sizeof(WideSmem) + 1024;
  static OncePerDevice attr_set;
  if (!attr_set.run([&] { return cudaFuncSetAttribute(gemm_fp8_wide_kernel<GROUPED, BIAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }))
    return AMCT_ERR_CUDA;
  // row tiles per rasterisation group: as many as keep the group's rows of A near 32 MB, a quarter of L2
  const int64_t g = (32LL << 20) / (p.k * kBlock);
  p.group_m = (int)(g < 4 ? 4 : g > 64 ? 64 : g);
  const int64_t tiles_n = (p.n + kWideN - 1) / kWideN;
  const int64_t row_tiles = (p.m + kBlock - 1) / kBlock + (GROUPED ? (p.experts < p.m ? p.experts : p.m) : 0);
  const int64_t most = row_tiles * tiles_n;
  if (most > 0x7fffffffLL) return AMCT_ERR_UNSUPPORTED;
  gemm_fp8_wide_kernel<GROUPED, BIAS><<<(unsigned)(most < sms ? most : sms), kWideThreads, smem, st>>>(ma, mb, p);
  AMCT_CHECK_LAUNCH();
  return AMCT_OK;
}

template <int NT, bool GROUPED>
static int launch_narrow(const void* a, const void* b, int64_t ld_a, int64_t ld_b, int64_t rows_b, const Params& p, int sms, cudaStream_t st) {
  CUtensorMap mw, mx;
  int rc = make_map(&mw, b, rows_b, p.k, ld_b, kBlock);
  if (rc != AMCT_OK) return rc;
  rc = make_map(&mx, a, p.m, p.k, ld_a, NT);
  if (rc != AMCT_OK) return rc;
  const size_t smem = sizeof(NarrowSmem<NT>) + 1024;
  static OncePerDevice attr_set;
  if (!attr_set.run([&] { return cudaFuncSetAttribute(gemm_fp8_narrow_kernel<NT, GROUPED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }))
    return AMCT_ERR_CUDA;
  const int64_t tiles_n = (p.n + kBlock - 1) / kBlock;
  // grouped: no more row tiles than this, however the rows are spread over the experts
  const int64_t row_tiles = GROUPED ? (p.experts < p.m ? p.experts : p.m) + p.m / NT : (p.m + NT - 1) / NT;
  const int64_t tiles = row_tiles * tiles_n;
  const int64_t num_kb = (p.k + kBlock - 1) / kBlock;
  int splits = 1;                                // K split until every SM has its CTAs, four K blocks left for each
  while (splits < kMaxSplits && tiles * splits * 2 <= narrow_ctas<NT>() * sms && num_kb >= splits * 2 * 4) splits *= 2;
  if (tiles * splits > 0x7fffffffLL) return AMCT_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * splits), 1, 1);
  cfg.blockDim = dim3(narrow_threads<NT>(), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, gemm_fp8_narrow_kernel<NT, GROUPED>, mw, mx, p, splits) != cudaSuccess) {
    cudaGetLastError();
    return AMCT_ERR_CUDA;
  }
  AMCT_CHECK_LAUNCH();
  return AMCT_OK;
}

template <bool GROUPED>
static int launch(const void* a, const void* b, int64_t ld_a, int64_t ld_b, int64_t rows_b, const Params& p, cudaStream_t st) {
  const int sms = sm_count();
  if (sms <= 0) return AMCT_ERR_CUDA;
  // Rows that share a weight: all of them, or an expert's on average.  Up to 64 the narrow kernel is ahead whatever the
  // weight (64 x 14336 x 4096: 20.6 us against 22.5; 48 x 4096 x 7168: 14 against 32).  Beyond, its 128-token form is ahead
  // only while it can split K, that is while its tiles fill at most half the SMs (256 x 4096 x 7168: 26.7 us against 34.4;
  // one split, 128 x 14336 x 4096: 28.7 against 24.8; 512 x 4096 x 7168: 43 against 35).
  const int64_t rows = GROUPED ? (p.m + p.experts - 1) / p.experts : p.m;
  if (rows <= 16) return launch_narrow<16, GROUPED>(a, b, ld_a, ld_b, rows_b, p, sms, st);
  if (rows <= 32) return launch_narrow<32, GROUPED>(a, b, ld_a, ld_b, rows_b, p, sms, st);
  if (rows <= 64) return launch_narrow<64, GROUPED>(a, b, ld_a, ld_b, rows_b, p, sms, st);
  const int64_t row_tiles = GROUPED ? (p.experts < p.m ? p.experts : p.m) + p.m / 128 : (p.m + 127) / 128;
  if (row_tiles * ((p.n + kBlock - 1) / kBlock) * 2 <= sms) return launch_narrow<128, GROUPED>(a, b, ld_a, ld_b, rows_b, p, sms, st);
  if constexpr (!GROUPED) {
    if (p.bias_kind != AMCT_BIAS_NONE) return launch_wide<false, true>(a, b, ld_a, ld_b, rows_b, p, sms, st);
  }
  return launch_wide<GROUPED, false>(a, b, ld_a, ld_b, rows_b, p, sms, st);
}

static int check(const void* a, int64_t ld_a, const float* sa, const void* b, int64_t ld_b, const float* sb, int64_t m, int64_t n,
                 int64_t k, const void* out, int out_kind, int64_t ld_out) {
  if (m < 0 || n < 0 || k <= 0 || ld_a < k || ld_b < k || ld_out < n) return AMCT_ERR_ARG;
  if (out_kind < AMCT_GEMM_OUT_F32 || out_kind > AMCT_GEMM_OUT_BF16) return AMCT_ERR_ARG;
  if (m == 0 || n == 0) return AMCT_OK;
  if (!a || !b || !sa || !sb || !out) return AMCT_ERR_ARG;
  if (m > 0x7fffff00LL || n > 0x7fffff00LL || k > 0x7fffff00LL) return AMCT_ERR_UNSUPPORTED;     // tensor-map coordinates
  if (!aligned16(a) || !aligned16(b) || ld_a % 16 != 0 || ld_b % 16 != 0) return AMCT_ERR_ALIGN;
  const uintptr_t size = out_kind == AMCT_GEMM_OUT_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(out) % size != 0) return AMCT_ERR_ALIGN;
  return AMCT_OK;
}

}  // namespace f8g
}  // namespace amct

extern "C" int amct_gemm_fp8_block(const void* a, const float* a_scale, int64_t a_scale_stride_row, int64_t a_scale_stride_k,
                                   const void* b, const float* b_scale, int64_t b_scale_stride_row, int64_t b_scale_stride_k,
                                   int64_t m, int64_t n, int64_t k, int64_t ld_a, int64_t ld_b, const void* bias, int bias_kind,
                                   void* out, int out_kind, int64_t ld_out, int* status, void* stream) {
  using namespace amct::f8g;
  const int rc = check(a, ld_a, a_scale, b, ld_b, b_scale, m, n, k, out, out_kind, ld_out);
  if (rc != AMCT_OK) return rc;
  if (bias_kind != AMCT_BIAS_NONE && (bias_kind < AMCT_BIAS_F32 || bias_kind > AMCT_BIAS_BF16 || (n > 0 && !bias))) return AMCT_ERR_ARG;
  if (m == 0 || n == 0) return AMCT_OK;
  Params p{};
  p.m = m; p.n = n; p.k = k;
  p.sa = a_scale; p.sa_row = a_scale_stride_row; p.sa_k = a_scale_stride_k;
  p.sb = b_scale; p.sb_row = b_scale_stride_row; p.sb_k = b_scale_stride_k;
  p.bias = bias; p.bias_kind = bias_kind; p.out = out; p.out_kind = out_kind; p.ld_out = ld_out; p.status = status;
  return launch<false>(a, b, ld_a, ld_b, n, p, (cudaStream_t)stream);
}

extern "C" int amct_gemm_fp8_block_grouped(const void* a, const float* a_scale, int64_t a_scale_stride_row, int64_t a_scale_stride_k,
                                           const int32_t* offsets, int experts, const void* b, const float* b_scale,
                                           int64_t b_scale_stride_expert, int64_t b_scale_stride_row, int64_t b_scale_stride_k,
                                           int64_t m, int64_t n, int64_t k, int64_t ld_a, int64_t ld_b, void* out, int out_kind,
                                           int64_t ld_out, int* status, void* stream) {
  using namespace amct::f8g;
  if (experts <= 0) return AMCT_ERR_ARG;
  const int rc = check(a, ld_a, a_scale, b, ld_b, b_scale, m, n, k, out, out_kind, ld_out);
  if (rc != AMCT_OK) return rc;
  if (m == 0 || n == 0) return AMCT_OK;
  if (!offsets) return AMCT_ERR_ARG;
  if (experts > kMaxExperts || n > 0x7fffff00LL / experts) return AMCT_ERR_UNSUPPORTED;
  Params p{};
  p.m = m; p.n = n; p.k = k;
  p.sa = a_scale; p.sa_row = a_scale_stride_row; p.sa_k = a_scale_stride_k;
  p.sb = b_scale; p.sb_expert = b_scale_stride_expert; p.sb_row = b_scale_stride_row; p.sb_k = b_scale_stride_k;
  p.out = out; p.out_kind = out_kind; p.ld_out = ld_out; p.status = status;
  p.offsets = offsets; p.experts = experts;
  return launch<true>(a, b, ld_a, ld_b, (int64_t)experts * n, p, (cudaStream_t)stream);
}
