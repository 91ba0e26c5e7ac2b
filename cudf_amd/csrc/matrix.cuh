// Shared by the kernels that feed the matrix cores (linear, attention): fragments, loads that write LDS, and their waits.
#pragma once

#include "encoder.cuh"

#include <utility>

namespace nvtext_amd {

constexpr uint32_t kFar = 0x80000000u;  // an offset outside every buffer, whatever is added for a row of the tile

typedef float f32x4_t __attribute__((ext_vector_type(4)));
template <typename T>
using Fragment = T __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
using LdsBytes = __attribute__((address_space(3))) char*;

// The same in every lane, and known to be.
__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ const char* uniform(const char* p)
{
  uint64_t const v    = reinterpret_cast<uint64_t>(p);
  uint32_t const low  = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v)), high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<const char*>(static_cast<uint64_t>(high) << 32 | low);
}

// 16 bytes a lane from base + offset to 16 bytes a lane from `to` on; zeros where the offset is not less than `range`.  Written out: the
// compiler would wait for loads that it knows to write LDS before every transposing read of LDS (a product of which one operand
// is read that way took 153 us instead of 118).  It has no register as a result, so it is waited for by stage_barrier alone.
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t range, LdsBytes to, uint32_t offset)
{
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  uint64_t const address = reinterpret_cast<uint64_t>(base);
  // a buffer: address, no stride, length, plain 32-bit data
  u32x4 const buffer = {static_cast<uint32_t>(address), static_cast<uint32_t>(address >> 32) & 0xffffu, range, 0x00027000u};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to))), "v"(offset), "s"(buffer)
               : "memory");  // (m0 is set wherever the compiler uses it itself)
}

// The same with 4 bytes a lane.
__device__ __forceinline__ void load_words_to_lds(const char* base, uint32_t range, LdsBytes to, uint32_t offset)
{
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  uint64_t const address = reinterpret_cast<uint64_t>(base);
  u32x4 const buffer = {static_cast<uint32_t>(address), static_cast<uint32_t>(address >> 32) & 0xffffu, range, 0x00027000u};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to))), "v"(offset), "s"(buffer) : "memory");
}

// All wavefronts have come here, their reads of LDS are done, and of the loads of each all but the last N.  (Written out: a fence in
// front of the barrier would wait for all loads, because they write LDS.)
template <int N>
__device__ __forceinline__ void stage_barrier()
{
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
  asm volatile("s_barrier" ::: "memory");
}

// f(0), ... f(N - 1) with the numbers as constants, so that arrays that they index stay in registers.
template <typename F, int... I>
__device__ __forceinline__ void for_each(std::integer_sequence<int, I...>, F&& f)
{
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void for_each(F&& f)
{
  for_each(std::make_integer_sequence<int, N>{}, f);
}

}  // namespace nvtext_amd
