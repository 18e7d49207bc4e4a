// Device-side helpers of the attention kernels that stream pages straight to LDS
// and join partial results of several blocks.
#pragma once

#include "tmc_device.hpp"

namespace tmc {
namespace {

static __device__ __align__(16) unsigned s_zero_row[4];  // what absent positions read

// A matrix product's result may be read by vector instructions only some wait
// states later.  The compiler puts them in within a block of code, but hipcc
// 7.2 left them out where a branch follows the product: the scores' maximum
// was then taken of old registers.
template <typename T> __device__ __forceinline__ void settle(T& result) {
  asm volatile("s_nop 15" : "+v"(result));
}

template <int N> __device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// Maximum over lanes l, l + 16, l + 32, l + 48.
__device__ __forceinline__ float max_of_groups(float v) {
  const unsigned x = __builtin_bit_cast(unsigned, v);
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const unsigned a0 = a[0], a1 = a[1];
  v = fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
  const unsigned y = __builtin_bit_cast(unsigned, v);
  const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  const unsigned b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// Two floats that other blocks read, and two of theirs: at agent scope.
__device__ __forceinline__ void store_pair(float* to, float a, float b) {
  const float2 v = {a, b};
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(to),
                     __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_pair(const float* from) {
  return __builtin_bit_cast(
      float2, __hip_atomic_load(reinterpret_cast<const unsigned long long*>(from),
                                __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
// A greatest score that is infinite, as where all are NaN or -inf, leaves no
// result but NaN, with weights of any type.
__device__ __forceinline__ bool finite(float top) { return fabsf(top) < INFINITY; }

}  // namespace
}  // namespace tmc
