// What the attention kernels share (gfx950): 64-row tiles of head dim 64 in LDS, their swizzles, the
// LDS-DMA that fills them and the transposing reads.
#pragma once

#include "common.h"

namespace i2pc {
namespace attn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint16_t bf16_t;

constexpr int kKV = 64;   // keys per tile
constexpr int kTileBytes = kKV * 64 * 2;   // 8 KiB (K tile and V^T tile each)

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  // one v_cvt_pk_bf16_f32 for the pair (RNE), no shift/or repacking
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

// V image (read by transposed reads): 16-B chunk c of row r at c ^ v_swz(r), which keeps them conflict-free
__device__ __forceinline__ int v_swz(int row) { return ((row >> 1) & 1) << 2; }
// K image: 16-B chunk c of key row r at c ^ ((r >> 1) & 7).  A ds_read_b128 serves 16 lanes per LDS
// cycle (lane groups {0-3,12-15,20-27}, {4-11,16-19,28-31} and their +32 twins); a group's 16 keys
// fall into 8 even and 8 odd rows, the parity picks the 128-B half of the 256-B bank row, and
// (r >> 1) & 7 is a bijection on each parity class of a group -- conflict-free.  (With r & 7 keys 20-27
// meet the chunks of keys 0-3 / 12-15: every K read is 2-way conflicted.)
__device__ __forceinline__ int k_swz(int row) { return (row >> 1) & 7; }

typedef short v4s __attribute__((ext_vector_type(4)));

// 16 B per lane global -> LDS at lds_base + 16 * lane (buffer_load ... lds), issued by inline asm.
// Through __builtin_amdgcn_raw_ptr_buffer_load_lds the compiler sees an LDS write it cannot prove
// disjoint from the current tile's ds_reads, so it put s_waitcnt vmcnt(3..0) in front of this tile's
// QK^T MFMAs -- each tile waited for the NEXT tile's K / V to land and the prefetch hid nothing.  The
// kernel orders the DMA itself: vmcnt(0) + barrier before a buffer is read.  M0 carries the LDS base
// and is declared clobbered, so the compiler saves / restores any M0 value of its own around it; the
// s_nop is gfx9's wait state between the write of M0 and the LDS-DMA that reads it.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, uint32_t lds_base, uint32_t voff, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(lds_base), "v"(voff), "s"(rs), "s"(soff)
               : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

__device__ __forceinline__ v4s tr_read(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(p));
}

}  // namespace attn
}  // namespace i2pc
