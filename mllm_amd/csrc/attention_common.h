// What the attention kernels share: operands of the matrix instructions, maxima over lanes, fp32 numbers as bf16 parts.
#pragma once
#include "item8.h"

namespace mllmhip {

typedef short at_s16x4 __attribute__((ext_vector_type(4)));
typedef short at_s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef float at_f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float larger(float x, float y) { return __builtin_elementwise_maximum(x, y); }
template <int N>  // the larger of a lane's and that of the lane N away
__device__ __forceinline__ float across(float v) {
  const u32x2 r = N == 16 ? lanes16(__float_as_uint(v)) : lanes32(__float_as_uint(v));
  return larger(__uint_as_float(r.x), __uint_as_float(r.y));
}
// 8 bf16 of a register quad as an operand
__device__ __forceinline__ at_bf16x8 frag(u32x4 v) { return __builtin_bit_cast(at_bf16x8, v); }
__device__ __forceinline__ at_f32x4 mma(at_bf16x8 x, at_bf16x8 y, at_f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, acc, 0, 0, 0); }

// Two numbers as three bf16 each, cut off after 8 bits of what is left: together they are the numbers.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const uint32_t xh = __float_as_uint(x), yh = __float_as_uint(y);
  const float x1 = x - __uint_as_float(xh & 0xffff0000u), y1 = y - __uint_as_float(yh & 0xffff0000u);
  const uint32_t xm = __float_as_uint(x1), ym = __float_as_uint(y1);
  const float x2 = x1 - __uint_as_float(xm & 0xffff0000u), y2 = y1 - __uint_as_float(ym & 0xffff0000u);
  hi = __builtin_amdgcn_perm(yh, xh, 0x07060302u);  // the high halves of both
  mid = __builtin_amdgcn_perm(ym, xm, 0x07060302u);
  lo = __builtin_amdgcn_perm(__float_as_uint(y2), __float_as_uint(x2), 0x07060302u);
}
__device__ __forceinline__ float finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? 0.f : x; }
// whether one of two bf16 is infinite or no number
__device__ __forceinline__ bool odd_pair(uint32_t v) { return ((v & 0x7f80u) == 0x7f80u) | ((v & 0x7f800000u) == 0x7f800000u); }
__device__ __forceinline__ uint32_t finite_pair(uint32_t v) {
  return ((v & 0x7f80u) == 0x7f80u ? 0u : v & 0xffffu) | ((v & 0x7f800000u) == 0x7f800000u ? 0u : v & 0xffff0000u);
}

// Eight elements of a query as an operand: bf16 as they are, fp32 as three parts of 8 bits each (what is infinite or no number: all in the first)
template <bool F32>
__device__ __forceinline__ void item_parts(const Item8<F32 ? MLLM_HIP_F32 : MLLM_HIP_BF16>& it, at_bf16x8 (&part)[F32 ? 3 : 1]) {
  if constexpr (!F32) {
    part[0] = frag(it.r[0]);
  } else {
    float v[8];
    item_to_f32<MLLM_HIP_F32>(it, v);
    uint32_t w[3][4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float x = v[2 * j], y = v[2 * j + 1];
      split2(finite(x), finite(y), w[0][j], w[1][j], w[2][j]);
      w[0][j] = (finite(x) == x ? w[0][j] & 0xffffu : f32_to_bf16(x)) | (finite(y) == y ? w[0][j] & 0xffff0000u : (uint32_t)f32_to_bf16(y) << 16);
    }
#pragma unroll
    for (int p = 0; p < 3; p++) part[p] = frag(u32x4{w[p][0], w[p][1], w[p][2], w[p][3]});
  }
}
// elements at .. at + 7, zeros where not `live`
template <bool F32>
__device__ __forceinline__ void query_parts(const void* q, int64_t at, bool live, at_bf16x8 (&part)[F32 ? 3 : 1]) {
  Item8<F32 ? MLLM_HIP_F32 : MLLM_HIP_BF16> it = {};
  if (live) item_load<F32 ? MLLM_HIP_F32 : MLLM_HIP_BF16>(q, at, it);
  item_parts<F32>(it, part);
}

}  // namespace mllmhip
