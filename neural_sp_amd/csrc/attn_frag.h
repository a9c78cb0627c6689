// attn_frag.h -- operand fragments shared by the decoder's attention kernels (paged_attn.hip, cross_attn.hip).
//
// Both element types run the same algorithms on 16 x 16 matrix-core tiles:
//   bf16  v_mfma_f32_16x16x32_bf16   one instruction contracts 32 elements, a lane holds 8 of them (16 bytes)
//   fp32  v_mfma_f32_16x16x4_f32     one instruction contracts 4 elements, a lane holds 1
// Lane l = r + 16 g.  An operand's row (or column) is r, the result's column is r and its rows are 4 g + e, e = 0..3.
//
// "chunk" = 16 consecutive bytes of a row.  A product over the head size takes chunk 4 s + g of row r per lane and step:
// for bf16 that is the instruction's own order; for fp32 the four elements of a chunk go to four instructions, the e-th of
// which contracts elements 16 s + 4 g + e over g -- any order will do as long as both operands use it.
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(4))) unsigned int nsp_u32x4;

template <typename T>
struct AttnElem;
template <>
struct AttnElem<float> {
  typedef f32x4 chunk;
  static constexpr int CE = 4;   // elements of a chunk
  __device__ static __forceinline__ chunk zero() { return f32x4{0.f, 0.f, 0.f, 0.f}; }
  __device__ static __forceinline__ f32x4 mma(const chunk& a, const chunk& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ static __forceinline__ float to_f32(float v) { return v; }
  __device__ static __forceinline__ float from_f32(float v) { return v; }
};
template <>
struct AttnElem<__bf16> {
  typedef bf16x8 chunk;
  static constexpr int CE = 8;
  __device__ static __forceinline__ chunk zero() {
    const nsp_u32x4 z = {0u, 0u, 0u, 0u};
    return __builtin_bit_cast(bf16x8, z);
  }
  __device__ static __forceinline__ f32x4 mma(const chunk& a, const chunk& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ float to_f32(__bf16 v) { return (float)v; }
  __device__ static __forceinline__ __bf16 from_f32(float v) { return (__bf16)v; }
};

constexpr float NSP_LOG2E = 1.4426950408889634f;

// (IEEE maximum: a NaN wins, and unlike fmaxf it needs no quieting of its operands first -- one instruction, or half of one)
__device__ __forceinline__ float attn_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// max / sum over the four lanes that share r (lanes r, r + 16, r + 32, r + 48): one lane-swap instruction per step
__device__ __forceinline__ float attn_max4(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = attn_max(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return attn_max(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float attn_sum4(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
