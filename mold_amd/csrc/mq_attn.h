// mq_attn.h — what the attention kernels share: the scale they take, the LDS DMA and its
// barrier, the exchange between a wave's halves, and the rounding of a pair to bf16.
#pragma once

#include "mq_kernels.h"

namespace mq {
namespace {

typedef __attribute__((address_space(3))) char lds_char;
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504f;

// What a row's running maximum starts at: a score below which scale (times log2(e)) s is no
// finite f32, so that the maximum times the scale always is one, also while every score
// seen is minus infinity: each then weighs 2^-inf, and not 2^(-inf + inf).  The last bits
// are room for the division's and the product's roundings.
inline float least_score(float scale) {
  const float s = scale * kLog2e;
  return s > 1.f ? -__FLT_MAX__ * (1.f - 0x1p-22f) / s : -__FLT_MAX__;
}

// Scales that the kernels take: scale log2(e) is a finite f32 too.
inline bool takes_scale(float scale) { return scale > 0.f && scale * kLog2e <= __FLT_MAX__; }

// 16 bytes per lane from base + off straight into LDS (lane i at lds + 16 i);
// base and lds are wave-uniform.  Read only after block_barrier.
__device__ __forceinline__ void dma16(const char *base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds)
               : "memory", "m0");
}

// This wave's DMA has landed and its LDS reads are complete; then every wave arrives.
__device__ __forceinline__ void block_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) expcnt(7) lgkmcnt(0)
  asm volatile("s_barrier" ::: "memory");
}

// The value combined with lane ^ 32's.
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_add(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 p = __builtin_convertvector((f32x2){a, b}, bf16x2);
  uint32_t u;
  __builtin_memcpy(&u, &p, 4);
  return u;
}

}  // namespace
}  // namespace mq
