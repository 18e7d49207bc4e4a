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

// The operands of one step out of LDS, waits included: the compiler would let
// such reads wait for every load to LDS in flight.
template <int D, int STEP, int OFFSET, int PAGE_OFFSET>
__device__ __forceinline__ void read_keys(const unsigned (&at)[D / 32], unsigned page_at,
                                          h8 (&k)[STEP / 16][D / 32], int& page) {
  static_assert((D == 128 && STEP == 16) || (D == 64 && STEP == 32), "four operands a step");
  if constexpr (D == 128) {
    asm volatile(
        "ds_read_b32 %4, %9 offset:%11\n\t"
        "ds_read_b128 %0, %5 offset:%10\n\tds_read_b128 %1, %6 offset:%10\n\t"
        "ds_read_b128 %2, %7 offset:%10\n\tds_read_b128 %3, %8 offset:%10\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[0][2]), "=&v"(k[0][3]), "=&v"(page)
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(page_at), "n"(OFFSET),
          "n"(PAGE_OFFSET)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b32 %4, %7 offset:%10\n\t"
        "ds_read_b128 %0, %5 offset:%8\n\tds_read_b128 %1, %6 offset:%8\n\t"
        "ds_read_b128 %2, %5 offset:%9\n\tds_read_b128 %3, %6 offset:%9\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[1][0]), "=&v"(k[1][1]), "=&v"(page)
        : "v"(at[0]), "v"(at[1]), "v"(page_at), "n"(OFFSET), "n"(OFFSET + 32 * D),
          "n"(PAGE_OFFSET)
        : "memory");
  }
}

// V^T, lane (j, g): dims 16 t + j, positions 4g .. 4g+3 of the step's first 16
// (v[0]) and, D = 64, of its last 16 (v[1]).
template <int D, int STEP, int OFFSET>
__device__ __forceinline__ void read_values(const unsigned (&at)[D / 16], h4 (&v)[STEP / 16][D / 16]) {
  if constexpr (D == 128) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%16\n\tds_read_b64_tr_b16 %1, %9 offset:%16\n\t"
        "ds_read_b64_tr_b16 %2, %10 offset:%16\n\tds_read_b64_tr_b16 %3, %11 offset:%16\n\t"
        "ds_read_b64_tr_b16 %4, %12 offset:%16\n\tds_read_b64_tr_b16 %5, %13 offset:%16\n\t"
        "ds_read_b64_tr_b16 %6, %14 offset:%16\n\tds_read_b64_tr_b16 %7, %15 offset:%16\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[0][2]), "=&v"(v[0][3]), "=&v"(v[0][4]),
          "=&v"(v[0][5]), "=&v"(v[0][6]), "=&v"(v[0][7])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]),
          "v"(at[7]), "n"(OFFSET)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %9 offset:%12\n\t"
        "ds_read_b64_tr_b16 %2, %10 offset:%12\n\tds_read_b64_tr_b16 %3, %11 offset:%12\n\t"
        "ds_read_b64_tr_b16 %4, %8 offset:%13\n\tds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
        "ds_read_b64_tr_b16 %6, %10 offset:%13\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[0][2]), "=&v"(v[0][3]), "=&v"(v[1][0]),
          "=&v"(v[1][1]), "=&v"(v[1][2]), "=&v"(v[1][3])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(OFFSET), "n"(OFFSET + 32 * D)
        : "memory");
  }
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
