// What the attention kernels share (lcsa_attn.hip, packed_attn.hip): exchanges between a wave's halves, tiles copied
// from buffers straight into LDS.
#pragma once
#include "common.hpp"

namespace fvsr {

// the larger, and the sum, of lanes l and l + 32 (in both)
__device__ __forceinline__ float pair_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// >= 19 wait states after the last MFMA of a walk (the compiler also inserts what it needs)
__device__ __forceinline__ void acc_drain() { asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory"); }

typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) char lds_char;

// s_waitcnt vmcnt(n) lgkmcnt(0) (gfx9 encoding: vmcnt bits [3:0] and [15:14], expcnt [6:4], lgkmcnt [11:8])
#define FVSR_WAIT_VM_LGKM0(n) __builtin_amdgcn_s_waitcnt(((n) & 15) | ((((n) >> 4) & 3) << 14) | (7 << 4))

// 16 bytes per lane from a buffer straight into LDS at lds_base + OFF + 16 * lane. Issued as inline assembly so the
// compiler does not order every later LDS read behind it: the kernel orders the copies itself (vmcnt + barrier).
// M0 is written without a clobber declaration (the compiler reserves it); nothing else in these kernels uses M0. It
// is loaded with s_mov_b32 from an address computed outside the asm. GFX9 requires one wait state between an SALU
// write of M0 and an LDS DMA that reads it; the compiler inserts it for its own code but not inside an asm
// statement, so the s_nop is written out.
// The row's offset `voff` and the block's offset `boff` are added into the one VGPR offset (the SGPR offset is 0):
// the raw buffer's range check covers the VGPR offset and the instruction offset, not the SGPR offset, so only an
// offset held there makes a row past the buffer (a ragged last block, a listed index outside [0, nk), the tiles past
// the end of the walk, whose block offset is the buffer's size) load zeros without touching memory.
template <int OFF>
__device__ __forceinline__ void dma16(u32x4 rsrc, uint32_t lds_base, int voff, int boff) {
  const uint32_t off = (uint32_t)voff + (uint32_t)boff;   // voff holds the head's offset, inside the buffer: < 2^32
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds_base + OFF),
               "v"(off), "s"(rsrc));
}

__device__ __forceinline__ u32x4 buffer_rsrc(const void* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)base;
  return u32x4{(uint32_t)a, (uint32_t)(a >> 32) & 0xffffu, bytes, 0x00020000u};
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}

}  // namespace fvsr
