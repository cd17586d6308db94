// ss_mfma.h - operand types and helpers of the MFMA attention kernels (internal).
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>

#include "ss_device.h"

namespace ssk {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef __attribute__((address_space(3))) v4s* lds_v4s_t;
typedef __attribute__((address_space(1))) void* gbl_ptr_t;

// the softmax of both attention kernels (ss_flash.h says why)
constexpr float kLog2e = 1.44269504088896340736f, kLog2eLow = 1.92596299e-8f;   // log2 e = their sum
constexpr float kPExp = 12.0f, kPScale = 4096.0f;   // P is held times 2^12
constexpr float kLag = 3.0f;        // the running maximum's lag (base 2)
constexpr float kLagX = 2.0f;       // int8: the lag of the exponent of weight times V scale

// the value of the lane with the same query row (lane ^ 32) joined to this one's
__device__ __forceinline__ float max_pair(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_pair(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// 2^e of a whole number (or -inf: 0)
__device__ __forceinline__ float pow2(float e) { return ldexpf(1.0f, (int)fmaxf(e, -200.f)); }

// hi + lo = v (to 2^-23 of |v| for normal values) as two fp16 vectors
__device__ __forceinline__ void split8(const float* v, v8h& hi, v8h& lo) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const _Float16 h = (_Float16)v[i];
    hi[i] = h;
    lo[i] = (_Float16)(v[i] - (float)h);
  }
}

// 8 int8 codes -> fp16, exact: 1024 + (code + 128) by placing the byte, less 1152
__device__ __forceinline__ v4u codes8(uint32_t lo, uint32_t hi) {
  const v2h off = {(_Float16)1152.f, (_Float16)1152.f};
  v4u r;
  lo ^= 0x80808080u;
  hi ^= 0x80808080u;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u)) - off);
  r[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u)) - off);
  r[2] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u)) - off);
  r[3] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)) - off);
  return r;
}

}  // namespace
}  // namespace ssk
