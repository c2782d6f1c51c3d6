// Global memory -> LDS without registers in between, for kernels in which one operand side streams through LDS.
#pragma once
#include <type_traits>
#include "common.h"

// A wavefront's load brings 64 pieces of 16 bytes to consecutive LDS places; which piece a lane fetches is free, so the
// tile's rows lie without padding and piece p of row r at p ^ lz_swz(r): conflict-free (4 cycles a wavefront instruction,
// 8 with rows 16 bytes apart) for the 16-byte row reads of a 32x32 operand and for the transposing reads.
// The loads are inline assembly that the compiler's wait counts do not know: the kernels wait by hand, for all but the
// loads of the last step (vector-memory operations complete in order).
template <int D>
__device__ __forceinline__ int lz_swz(int r) {
  return D == 128 ? (r & 3) << 2 | (r >> 2 & 3) : (r >> 1 & 1) << 2 | (r >> 2 & 3);
}
__device__ __forceinline__ unsigned long long lz_uniform(unsigned long long x) {
  return (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)x) |
         (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}
__device__ __forceinline__ unsigned lz_lds_addr(const unsigned char* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)p;
}
// (M0, which both statements set, is a register that the compiler never holds a variable in: it warns that naming it cannot
// preserve it.  Named, its own settings of M0 are not taken to last over the statement, which is what is wanted.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 64 pieces of 16 bytes, lane i's from base + off to lds + 16 i
__device__ __forceinline__ void lz_dma16(unsigned lds, unsigned off, unsigned long long base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
// 64 words, lane i's from addr to lds + 4 i
__device__ __forceinline__ void lz_dma4(unsigned lds, unsigned long long addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(addr) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void lz_landed() {  // all but the last N vector-memory operations
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ float lz_halves_sum(float x) {
  const hils_uint2v y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(y.x) + __uint_as_float(y.y);
}
__device__ __forceinline__ float lz_halves_max(float x) {
  const hils_uint2v y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(y.x), __uint_as_float(y.y));
}
// Steps 0 .. n-1, four a round: the buffers' numbers are constants, and so the LDS addresses fixed registers
// and immediate offsets.
template <typename F>
__device__ __forceinline__ void lz_walk(int n, F&& step) {
  for (int c = 0; c < n; c += 4) {
    step(c, std::integral_constant<int, 0>{});
    if (c + 1 < n) step(c + 1, std::integral_constant<int, 1>{});
    if (c + 2 < n) step(c + 2, std::integral_constant<int, 2>{});
    if (c + 3 < n) step(c + 3, std::integral_constant<int, 3>{});
  }
}
