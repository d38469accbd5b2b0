// Matrix products and their operands: what the attention kernels over paged caches share.
#pragma once

#include "ds355_common.h"

namespace ds355 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2eP = 1.44269504088896340736f;
constexpr float kLn2P = 0.69314718055994530942f;

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// The thread's index, opaque to the compiler: what a part of the loop derives from it is derived there
// again, instead of being kept in registers that the loop needs (spilled ones would be loaded in order
// behind the keys in flight).
__device__ __forceinline__ int fresh_thread() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// A value that is the same in all lanes, to the scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The kernel's one argument, read again, so that what a loop does not need takes no scalar registers in it.
template <typename Args>
__device__ __forceinline__ Args arguments() {
  static_assert(sizeof(Args) % 8 == 0);
  struct Words {
    uint64_t w[sizeof(Args) / 8];
  } words;
  typedef const __attribute__((address_space(4))) uint64_t* pointer;  // scalar loads
  pointer at = (pointer)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
#pragma unroll
  for (unsigned i = 0; i < sizeof(Args) / 8; ++i) words.w[i] = at[i];
  return __builtin_bit_cast(Args, words);
}

// ---------------------------------------------------------------------------------------------
// Matrix products: 32x32x16, A rows and B columns of 32, k-slot (lane / 32, e) = 8 (lane / 32) + e;
// result i of a lane is row 8 (i / 4) + 4 (lane / 32) + i % 4 of column lane % 32.
// ---------------------------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ f32x16 mfma32(u32x4 x, u32x4 y, f32x16 c) {
  if constexpr (DT == DS_BF16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0,
                                                   0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0,
                                                  0);
  }
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (DT == DS_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {static_cast<__bf16>(x), static_cast<__bf16>(y)};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 v = {static_cast<_Float16>(x), static_cast<_Float16>(y)};
    return __builtin_bit_cast(uint32_t, v);
  }
}

// Combines a lane's value with lane ^ 32's.
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

__device__ __forceinline__ bool not_finite2(uint32_t w, uint32_t exponent) {
  return (w & exponent) == exponent || (w & (exponent << 16)) == (exponent << 16);
}

// Where 16-byte piece `c` of staged value `t` lies (in pieces): the pieces of eight neighbouring keys
// are turned against each other by two, so that a transposing read (two pieces of four keys) touches
// different banks.
template <int D>
__device__ __forceinline__ int piece_at(int t, int c) {
  const int turn = D >= 128 ? 2 * (t & 7) : 2 * ((t >> 1) & 3);
  return t * (D / 8) + (c ^ turn);
}

// Key t's 16-byte piece c lies at place c ^ turn of its row, so that the reads of 16 neighbouring keys
// touch different banks.
template <int D>
__device__ __forceinline__ int key_turn(int t) {
  return D == 64 ? (t >> 1) & 7 : t & 15;
}

__device__ __forceinline__ uint64_t lane_value(uint64_t v, int i) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), i);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), i);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// 64 lanes' 16 bytes each from base + offset to 1 KiB of shared memory from to + PLUS on, a lane after the
// other.  The compiler does not know of the load: what reads that memory waits for it (wait_loads) before a
// barrier.  (It keeps nothing in m0 from one instruction to another.)
template <int PLUS>
__device__ __forceinline__ void load_lds(uint64_t base, uint32_t offset, uint32_t to) {
  asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3"
               :
               : "s"(to), "i"(PLUS), "v"(offset), "s"(base)
               : "memory", "scc");
}
template <int PLUS>
__device__ __forceinline__ void load_lds(uint64_t from, uint32_t to) {
  asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off"
               :
               : "s"(to), "i"(PLUS), "v"(from)
               : "memory", "scc");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }

typedef __attribute__((address_space(3))) char lds_char;
// A transposing read: lane l of 16 names key l / 4 and dimensions 4 (l % 4) .. + 3 and gets four keys of dimension l.
__device__ __forceinline__ u32x2 read_values(uint32_t at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_char*)(uintptr_t)at));
}

}  // namespace
}  // namespace ds355
