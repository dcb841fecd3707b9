// What moe_permute.cu and fp8_block_quant.cu use beyond cuda_emu.h.  TEST INFRASTRUCTURE ONLY.
#pragma once
#include "cuda_emu.h"

static inline void __syncwarp() {
  emu::ThreadState& s = emu::tls();
  s.block->warp[s.tid.x >> 5].wait();
}
// lanes of the warp that hold the same value; all 32 take part
static inline unsigned __match_any_sync(unsigned, int v) {
  unsigned mask = 0;
  const int lane = (int)(emu::tls().tid.x & 31u);
  for (int l = 0; l < 32; ++l)
    if ((int)emu::shfl_idx_bits((uint32_t)v, l) == v) mask |= 1u << l;
  (void)lane;
  return mask;
}
static inline int atomicAdd(int* p, int v) { return __atomic_fetch_add(p, v, __ATOMIC_SEQ_CST); }
static inline float __saturatef(float x) { return x > 0.f ? (x < 1.f ? x : 1.f) : 0.f; }
#define __expf(x) (std::exp((float)(x)))          // a name that the C library declares too
static inline float __fdividef(float a, float b) { return a / b; }
