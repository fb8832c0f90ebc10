// Rows staged in LDS by loads that bypass the registers, read with the matrix
// cores' operand layouts; for the kernels over a paged cache.
#pragma once

#include <utility>

#include "common.h"

namespace moba {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 16-byte pieces of a row stand in LDS at piece ^ swizzle_rows(row), so that the
// 16 rows which a wave's lanes read together fall into different banks.
template <int D>
__device__ inline int swizzle_rows(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }

// LDS reads of the staged rows by assembly, each block with its wait: ahead of
// reads that it knows, the compiler waits for every load to LDS under way, the
// next item's among them.
__device__ inline uint32_t lds_address(const uint16_t* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint16_t*)p));
}

__device__ inline int32_t read_word(const int32_t* p) {
  int32_t x;
  asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(x) : "v"(lds_address(reinterpret_cast<const uint16_t*>(p))) : "memory");
  return x;
}

// 16 bytes at LDS address at ^ X, and STEP, 2 STEP, .. bytes behind it. The
// exclusive or stands here so that a register holds one address, not one for
// every X.
template <int X, int STEP>
__device__ inline void read_rows(uint32_t at, u32x4 (&x)[1]) {
  uint32_t t;
  asm volatile("v_xor_b32 %1, %3, %2\n\t"
               "ds_read_b128 %0, %1\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(x[0]), "=&v"(t)
               : "v"(at), "n"(X)
               : "memory");
}
template <int X, int STEP>
__device__ inline void read_rows(uint32_t at, u32x4 (&x)[2]) {
  uint32_t t;
  asm volatile("v_xor_b32 %2, %4, %3\n\t"
               "ds_read_b128 %0, %2\n\t"
               "ds_read_b128 %1, %2 offset:%5\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(x[0]), "=&v"(x[1]), "=&v"(t)
               : "v"(at), "n"(X), "n"(STEP)
               : "memory");
}
template <int X, int STEP>
__device__ inline void read_rows(uint32_t at, u32x4 (&x)[3]) {
  uint32_t t;
  asm volatile("v_xor_b32 %3, %5, %4\n\t"
               "ds_read_b128 %0, %3\n\t"
               "ds_read_b128 %1, %3 offset:%6\n\t"
               "ds_read_b128 %2, %3 offset:%7\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(t)
               : "v"(at), "n"(X), "n"(STEP), "n"(2 * STEP)
               : "memory");
}
template <int X, int STEP>
__device__ inline void read_rows(uint32_t at, u32x4 (&x)[4]) {
  uint32_t t;
  asm volatile("v_xor_b32 %4, %6, %5\n\t"
               "ds_read_b128 %0, %4\n\t"
               "ds_read_b128 %1, %4 offset:%7\n\t"
               "ds_read_b128 %2, %4 offset:%8\n\t"
               "ds_read_b128 %3, %4 offset:%9\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(t)
               : "v"(at), "n"(X), "n"(STEP), "n"(2 * STEP), "n"(3 * STEP)
               : "memory");
}

// 16 bytes at at ^ X and STEP behind it, and the same at at ^ X ^ 32.
template <int X, int STEP>
__device__ inline void read_row_pairs(uint32_t at, u32x4 (&x)[4]) {
  uint32_t t, u;
  asm volatile("v_xor_b32 %4, %7, %6\n\t"
               "v_xor_b32 %5, %8, %6\n\t"
               "ds_read_b128 %0, %4\n\t"
               "ds_read_b128 %1, %4 offset:%9\n\t"
               "ds_read_b128 %2, %5\n\t"
               "ds_read_b128 %3, %5 offset:%9\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(t), "=&v"(u)
               : "v"(at), "n"(X), "n"(X ^ 32), "n"(STEP)
               : "memory");
}

// Eight elements of V^T for one MFMA operand: two transposing reads, each of
// four keys by 16 features per 16 lanes, at a ^ X and b ^ X; for feature tiles
// X and X + 64; AT bytes behind.
template <int X, int AT>
__device__ inline void read_transposed(uint32_t a, uint32_t b, u32x2 (&x)[4]) {
  uint32_t t, u;
  asm volatile("v_xor_b32 %4, %8, %6\n\t"
               "v_xor_b32 %5, %8, %7\n\t"
               "ds_read_b64_tr_b16 %0, %4 offset:%10\n\t"
               "ds_read_b64_tr_b16 %1, %5 offset:%10\n\t"
               "v_xor_b32 %4, %9, %6\n\t"
               "v_xor_b32 %5, %9, %7\n\t"
               "ds_read_b64_tr_b16 %2, %4 offset:%10\n\t"
               "ds_read_b64_tr_b16 %3, %5 offset:%10\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(t), "=&v"(u)
               : "v"(a), "v"(b), "n"(X), "n"(X ^ 64), "n"(AT)
               : "memory");
}

// 16 bytes from global memory straight to LDS: lane i's to `dst` + 16 i.
__device__ inline void load_to_lds(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(
      reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(src)),
      (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// Waits until at most N of the wave's vector memory operations are under way
// (they end in order). Loads to LDS count as such: a barrier alone does not
// wait for them.
template <int N>
__device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A barrier that waits for no vector memory (__syncthreads waits for every
// load to LDS under way): each wave waits for its own before.
__device__ inline void meet() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 4 bytes each: lane i's to `dst` + 4 i.
__device__ inline void load_word_to_lds(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(
      reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(src)),
      (__attribute__((address_space(3))) void*)dst, 4, 0, 0);
}

// f of 0, 1, .. as constants.
template <int... J, typename F>
__device__ inline void steps(std::integer_sequence<int, J...>, F&& f) {
  (f(std::integral_constant<int, J>{}), ...);
}

}  // namespace moba
