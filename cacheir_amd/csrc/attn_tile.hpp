// Pieces shared by the attention kernels that run 32 query vectors x 32 tokens per MFMA
// tile (K and V staged in LDS by DMA).
#pragma once

#include "common.hpp"

namespace cir {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;

// Transposing LDS read (ds_read_b64_tr_b16): 16 lanes read 4 token rows of 16 dims and each gets 4 tokens of one dim.
__device__ __forceinline__ f16x4 lds_read_tr(const uint8_t* p) {
  typedef __fp16 h4 __attribute__((ext_vector_type(4)));
  const h4 v = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4*)(p));
  return __builtin_bit_cast(f16x4, v);
}
// This wavefront's DMA has landed, then every wavefront's.  The wait is the builtin, not asm: the compiler counts it,
// and then puts no wait of its own (which would cover the next stage's DMA too) before the reads of the landed stage.
__device__ __forceinline__ void dma_wait_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x70);  // vmcnt(0), lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace cir
