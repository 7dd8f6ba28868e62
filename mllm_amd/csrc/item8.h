// Eight consecutive elements of an fp32 or bf16 tensor in a lane's registers: loads, conversion to fp32, stores.
#pragma once
#include "qcommon.h"

namespace mllmhip {

// ---- eight consecutive elements per lane ------------------------------------------------------------------------------
template <int XT>
struct Item8 {
  u32x4 r[XT == MLLM_HIP_F32 ? 2 : 1];
};
template <int XT>
__device__ __forceinline__ void item_load(const void* p, int64_t elem, Item8<XT>& it) {
  if (XT == MLLM_HIP_F32) {
    const u32x4* q = reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(p) + elem);
    it.r[0] = q[0];
    it.r[XT == MLLM_HIP_F32 ? 1 : 0] = q[1];
  } else {
    it.r[0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p) + elem);
  }
}
template <int XT>
__device__ __forceinline__ void item_to_f32(const Item8<XT>& it, float (&v)[8]) {
  if (XT == MLLM_HIP_F32) {
    const u32x4 a = it.r[0], b = it.r[XT == MLLM_HIP_F32 ? 1 : 0];
    v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
    v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
  } else {
    const uint32_t w[4] = {it.r[0].x, it.r[0].y, it.r[0].z, it.r[0].w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      v[2 * j + 0] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
}
// stores v in the tensor's type and leaves in v what a reader of the tensor will see (bf16: the rounded values)
template <int XT>
__device__ __forceinline__ void item_store(void* p, int64_t elem, float (&v)[8]) {
  if (XT == MLLM_HIP_F32) {
    u32x4* q = reinterpret_cast<u32x4*>(reinterpret_cast<float*>(p) + elem);
    q[0] = u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    q[1] = u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
  } else {
    u32x4 o = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
    *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(p) + elem) = o;
    const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      v[2 * j + 0] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
}

// Every head of the results has a place of its own, and where that is the place of x, it is that of the same head
inline bool own_places(const mllm_hip_heads& p, int64_t T) {
  const bool tokens = T > 1, heads = p.heads > 1;
  if ((tokens && !p.y_token_stride) || (heads && !p.y_head_stride)) return false;
  return p.x != p.y || !((tokens && p.x_token_stride != p.y_token_stride) || (heads && p.x_head_stride != p.y_head_stride));
}

}  // namespace mllmhip
