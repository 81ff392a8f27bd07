// 4-bit expert weights: format, layout and the device code that turns codes into bf16 operands.
//
// Format.  w[n, k] = q[n, k] * s[n, k / group], q in [-7, 7], group 32, 64 or 128.  The scale is the
// smallest number of 5 significant bits (at least 2^-126) that is >= amax / 7 of its group, so
// q (3 bits) times s (5 bits) has at most 8 significant bits: every weight is exactly a bf16 number.
// Rounding it up to 5 bits widens the step by up to a sixteenth (6.25%, 2% on average; to bf16's 8 bits it would
// be 0.8%); in exchange the weights enter the products, on any path, without a rounding of their own.
//
// Layout.  Rows come in tiles of 16, columns in blocks of 128 (both padded with zero weights), the
// blocks of a tile one after the other.  A block of a tile is 2 x 512 bytes; in the half h, lane
// l = 4 g + t of a warp owns 16 bytes = 4 words: row g and row g + 8 of the columns 64 h + 8 t .. + 7,
// then of the columns 64 h + 32 + 8 t .. + 7.  This is the order in which the lanes of a warp feed both
// the m16n8k16 product's first operand and a 16-lane store to tensor memory; the order of columns
// inside a product does not matter as long as x is read the same way.
// A word's nibble i holds the code + 8 of column 2 i, nibble i + 4 that of column 2 i + 1, the word
// rotated left by 3: field i of each half then sits on bits 3..6 after a rotation by 4 i, where it is
// the upper mantissa of a bf16 number with exponent 4 (0x4180): 16 + n, n = q + 8.
// The scales of a block are [8][128 / group][2] bf16: for g < 8 and each group of the block, rows g
// and g + 8.  A GLU weight's prepared row 2 j is gate row j and 2 j + 1 up row j (the interleaved
// order; a concatenated w1 is re-ordered when it is prepared).
#pragma once

#include "common.cuh"
#include "sonic_internal.h"

namespace smb {

// The constants come from registers the compiler cannot look into: with two immediates it would spend two
// instructions instead of one on the and-or.
struct Int4Magic {
  uint32_t mask, base;
  __device__ __forceinline__ Int4Magic() {
    asm volatile("mov.u32 %0, 0x00780078;" : "=r"(mask));
    asm volatile("mov.u32 %0, 0x41804180;" : "=r"(base));
  }
};

// Columns 2 i and 2 i + 1 of a word as two bf16 numbers 16 + n = q + 24.
__device__ __forceinline__ uint32_t int4_raw(const Int4Magic& c, uint32_t w, int i) {
  uint32_t r;
  const uint32_t v = i == 0 ? w : __funnelshift_r(w, w, 4 * i);
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(c.mask), "r"(c.base));  // (a & b) | c
  return r;
}

// The same times the scale: s (16 + n) - 24 s in one fused operation.  24 s has 7 significant bits and
// q s has 8 at most, so both the addend and the result are exact.
__device__ __forceinline__ uint32_t int4_scaled(const Int4Magic& c, uint32_t w, int i, __nv_bfloat162 s,
                                                __nv_bfloat162 m24s) {
  const uint32_t u = int4_raw(c, w, i);
  __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&u), s, m24s);
  return *reinterpret_cast<uint32_t*>(&r);
}

// Half `hi` of a scale word (row g: 0, row g + 8: 1) in both halves of a register, and -24 times it.
__device__ __forceinline__ __nv_bfloat162 int4_scale2(uint32_t w, int hi) {
  const uint32_t u = __byte_perm(w, 0, hi ? 0x3232 : 0x1010);
  return *reinterpret_cast<const __nv_bfloat162*>(&u);
}
__device__ __forceinline__ __nv_bfloat162 int4_m24(__nv_bfloat162 s) {
  return __hmul2(s, __floats2bfloat162_rn(-24.0f, -24.0f));
}

__device__ __forceinline__ float silu_mul(float gate, float up) { return __fdividef(gate, 1.0f + __expf(-gate)) * up; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int kBytes>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

}  // namespace smb
