// RMSNorm of every query and key head and their rotation by position, and the same on the way into a paged cache, for gfx950.
//
//   n = x * (w * rms),  rms = 1 / sqrt(mean over the head (x^2) + epsilon)      (as mllm_hip_rmsnorm; left out without a weight)
//   pair (a, b) number j of a head at position p:  a' = a cos - b sin,  b' = b cos + a sin,  angle = p * inv_freq[j]
//
// Everything is fp32 between the load and the one rounding of the store.  The angle is not: fp32 holds p * f of a far position to
// a tenth of a radian at best, so it is multiplied in fp64, reduced to a fraction of a turn there, and only that goes to fp32.
// A workgroup has one token: its cosines and sines are computed once into LDS (64 pairs of 128 wide heads) while the first heads
// are on their way from memory, and every head of the token uses them.  Per byte there is nothing else to do: bound by memory
// with many tokens, by the launch and two dependent loads with few.
#include "item8.h"

namespace mllmhip {

enum { ROPE_OUT = 0, ROPE_KEYS = 1, ROPE_VALUES = 2 };  // where a part's heads go: a tensor, the cache's keys, the cache's values
struct RopeGroup {
  const void* x;
  void* y;
  const float* w;
  int64_t x_token, x_head, y_token, y_head;
  int head0, kind;
};
struct RopeArgs {
  RopeGroup part[4];
  int nparts, heads, D, rot, passes, add_unit_offset;
  float eps;
  const int32_t* positions;
  const double* inv_freq;
  // the cache's addressing
  const int64_t* slots;
  int64_t page_stride, slot_stride, head_stride, slot_count;
  uint32_t page;
};

// G lanes per head of up to 8 * G elements, 256 / G heads of a token at a time
template <int XT, int G, bool NEXT>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  __shared__ float s_cos[256], s_sin[256];
  const int tid = threadIdx.x, lane = tid & 63, lg = tid % G, e = lg * 8;
  const int64_t t = blockIdx.x;
  const int half = a.rot / 2;
  int head = blockIdx.y * a.passes * (256 / G) + tid / G;
  // (selects between scalar registers: a part looked up by a lane's index would be loads in front of the first load)
  auto part_of = [&](int h) {
    RopeGroup g = a.part[0];
#pragma unroll
    for (int j = 1; j < 4; j++)
      if (j < a.nparts && h >= a.part[j].head0) g = a.part[j];
    return g;
  };
  auto load = [&](int h, Item8<XT>& it) {
    const RopeGroup g = part_of(h);
    if (h < a.heads && e < a.D) item_load<XT>(g.x, t * g.x_token + (h - g.head0) * g.x_head + e, it);
  };
  Item8<XT> it = {};
  load(head, it);
  const int64_t slot = a.slots ? a.slots[t] : -1;
  if (half > 0) {
    if (tid < half) {
      // turns in fp64: p * f is off by 2^-53 of itself, which at 2^20 radians is 1e-10
      double turn = (double)a.positions[t] * a.inv_freq[tid] * 0.15915494309189533577;
      turn -= rint(turn);
      float sn, cs;
      sincospif(2.0f * (float)turn, &sn, &cs);
      s_cos[tid] = cs;
      s_sin[tid] = sn;
    }
    __syncthreads();
  }
  for (int p = 0; p < a.passes; p++, head += 256 / G) {
    const int h = head;
    float v[8];
    item_to_f32<XT>(it, v);
    if (p + 1 < a.passes) load(h + 256 / G, it);
    if (h - tid / G >= a.heads) return;  // (no head of this workgroup is left)
    const bool live = h < a.heads && e < a.D;
    const RopeGroup g = part_of(h);
    if (!live) {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = 0.f;
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) ss = fmaf(v[j], v[j], ss);
    ss = group_sum<G>(ss);
    if (live && g.w) {
      const float rms = 1.0f / sqrtf(ss / (float)a.D + a.eps);
      const float4 w0 = *reinterpret_cast<const float4*>(g.w + e), w1 = *reinterpret_cast<const float4*>(g.w + e + 4);
      const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = v[j] * ((a.add_unit_offset ? w[j] + 1.0f : w[j]) * rms);
    }
    if (half > 0) {
      const bool turns = live && g.kind != ROPE_VALUES && e < a.rot;
      if (NEXT) {
        if (turns) {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float cs = s_cos[e / 2 + j], sn = s_sin[e / 2 + j], x = v[2 * j], y = v[2 * j + 1];
            v[2 * j] = x * cs - y * sn;
            v[2 * j + 1] = y * cs + x * sn;
          }
        }
      } else {  // the other half of the pairs is half / 8 lanes away
        const bool first = e < half;
        const int from = first ? lane + half / 8 : lane - half / 8, j0 = first ? e : e - half;
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = __shfl(v[j], from);
        if (turns) {
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float cs = s_cos[j0 + j], sn = s_sin[j0 + j];
            v[j] = first ? v[j] * cs - o[j] * sn : v[j] * cs + o[j] * sn;
          }
        }
      }
    }
    if (!live) continue;
    const int hh = h - g.head0;
    if (g.kind == ROPE_OUT) {
      item_store<XT>(g.y, t * g.y_token + hh * g.y_head + e, v);
    } else if (slot >= 0 && slot < a.slot_count) {
      const uint32_t page = (uint32_t)slot / a.page, at = (uint32_t)slot - page * a.page;
      item_store<MLLM_HIP_BF16>(g.y, page * a.page_stride + at * a.slot_stride + hh * a.head_stride + e, v);
    }
  }
}

static bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// a part as the kernel takes it: checks of the strides that 16-byte loads and stores need
static int rope_group(const mllm_hip_heads& p, int dtype, int head_dim, bool stored, RopeGroup& g) {
  const int wide = dtype == MLLM_HIP_F32 ? 4 : 2;
  if (!p.x || (stored && !p.y) || p.heads < 1) return MLLM_HIP_E_BADARG;
  if (p.heads > 65536) return MLLM_HIP_E_SHAPE;
  auto whole = [&](int64_t stride) { return stride * wide % 16 == 0; };
  if (!al16(p.x) || !whole(p.x_token_stride) || !whole(p.x_head_stride) || (p.weight && !al16(p.weight))) return MLLM_HIP_E_ALIGN;
  if (stored && (!al16(p.y) || !whole(p.y_token_stride) || !whole(p.y_head_stride))) return MLLM_HIP_E_ALIGN;
  g = RopeGroup{p.x, p.y, p.weight, p.x_token_stride, p.x_head_stride, p.y_token_stride, p.y_head_stride, 0, ROPE_OUT};
  return 0;
}

// Workgroups of a token: one for all of its heads while there are tokens to fill the chip, else one per 256 / G heads.
static const int64_t ROPE_FULL = 2048;

static int rope_launch(RopeArgs& a, int dtype, int64_t T, int head_dim, int rot_dim, int interleaved, int heads, hipStream_t st) {
  const int lanes = head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : head_dim <= 256 ? 32 : 64;
  const int all = (heads + 256 / lanes - 1) / (256 / lanes);
  a.heads = heads;
  a.D = head_dim;
  a.rot = rot_dim;
  a.passes = T * all <= ROPE_FULL ? 1 : all;
  const dim3 grid((unsigned)T, (unsigned)(all / a.passes));
#define ROPE(XT_, G_)                                                                                    \
  if (interleaved) hipLaunchKernelGGL((rope_kernel<XT_, G_, true>), grid, dim3(256), 0, st, a);          \
  else hipLaunchKernelGGL((rope_kernel<XT_, G_, false>), grid, dim3(256), 0, st, a)
#define ROPE_T(XT_)                \
  if (lanes == 8) { ROPE(XT_, 8); } \
  else if (lanes == 16) { ROPE(XT_, 16); } \
  else if (lanes == 32) { ROPE(XT_, 32); } \
  else { ROPE(XT_, 64); }
  if (dtype == MLLM_HIP_F32) {
    ROPE_T(MLLM_HIP_F32)
  } else {
    ROPE_T(MLLM_HIP_BF16)
  }
#undef ROPE_T
#undef ROPE
  return (int)hipGetLastError();
}

// what both calls check of the rotation
static int rope_checks(int dtype, int64_t T, int head_dim, const int32_t* positions, const double* inv_freq, int rot_dim) {
  if ((dtype != MLLM_HIP_F32 && dtype != MLLM_HIP_BF16) || T < 0 || head_dim < 1 || rot_dim < 0) return MLLM_HIP_E_BADARG;
  if (T && rot_dim && (!positions || !inv_freq)) return MLLM_HIP_E_BADARG;
  if (head_dim % 8 || head_dim > 512 || rot_dim > head_dim || rot_dim % 16 || T > 0x7fffffff) return MLLM_HIP_E_SHAPE;
  if (reinterpret_cast<uintptr_t>(positions) % 4 || reinterpret_cast<uintptr_t>(inv_freq) % 8) return MLLM_HIP_E_ALIGN;
  return 0;
}

}  // namespace mllmhip

using namespace mllmhip;

MLLM_API int mllm_hip_qk_norm_rope(int nparts, const mllm_hip_heads* parts, int dtype, int64_t T, int head_dim, float epsilon,
                                   int add_unit_offset, const int32_t* positions, const double* inv_freq, int rot_dim,
                                   int interleaved, void* stream) {
  if (nparts < 1 || nparts > 4 || !parts) return MLLM_HIP_E_BADARG;
  RC_RET(rope_checks(dtype, T, head_dim, positions, inv_freq, rot_dim));
  if (T == 0) return 0;  // (tensors without elements have no addresses)
  RopeArgs a = {};
  int heads = 0;
  for (int i = 0; i < nparts; i++) {
    RC_RET(rope_group(parts[i], dtype, head_dim, true, a.part[i]));
    a.part[i].head0 = heads;
    heads += parts[i].heads;
  }
  a.nparts = nparts;
  a.eps = epsilon;
  a.add_unit_offset = add_unit_offset;
  a.positions = positions;
  a.inv_freq = inv_freq;
  return rope_launch(a, dtype, T, head_dim, rot_dim, interleaved, heads, (hipStream_t)stream);
}

MLLM_API int mllm_hip_kv_append(const mllm_hip_heads* q, const mllm_hip_heads* k, const mllm_hip_heads* v, int dtype, int64_t T,
                                const mllm_hip_kv_cache* cache, const int64_t* slots, float epsilon, int add_unit_offset,
                                const int32_t* positions, const double* inv_freq, int rot_dim, int interleaved, void* stream) {
  if (!k || !v || !cache || !cache->k || !cache->v || (T && !slots) || cache->heads < 1 || cache->pages < 1 || cache->page_size < 1) return MLLM_HIP_E_BADARG;
  RC_RET(rope_checks(dtype, T, cache->head_dim, positions, inv_freq, rot_dim));
  if (k->heads != cache->heads || v->heads != cache->heads || cache->pages > 0x7fffffff / cache->page_size || cache->page_stride < 0 ||
      cache->slot_stride < 0 || cache->page_stride > 0x7fffffff || cache->slot_stride > 0x3fffffff / cache->page_size ||
      (cache->slot_stride == 0 && cache->page_size > 1))
    return MLLM_HIP_E_SHAPE;
  if (!al16(cache->k) || !al16(cache->v) || cache->page_stride % 8 || cache->slot_stride % 8 || cache->head_stride % 8 ||
      reinterpret_cast<uintptr_t>(slots) % 8)
    return MLLM_HIP_E_ALIGN;
  if (T == 0) return 0;
  RopeArgs a = {};
  RC_RET(rope_group(*k, dtype, cache->head_dim, false, a.part[0]));
  RC_RET(rope_group(*v, dtype, cache->head_dim, false, a.part[1]));
  a.part[0].y = cache->k;
  a.part[0].kind = ROPE_KEYS;
  a.part[1].y = cache->v;
  a.part[1].kind = ROPE_VALUES;
  a.part[1].w = nullptr;
  a.part[1].head0 = k->heads;
  int heads = k->heads + v->heads;
  a.nparts = 2;
  if (q) {
    RC_RET(rope_group(*q, dtype, cache->head_dim, true, a.part[2]));
    a.part[2].head0 = heads;
    heads += q->heads;
    a.nparts = 3;
  }
  a.eps = epsilon;
  a.add_unit_offset = add_unit_offset;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.slots = slots;
  a.page_stride = cache->page_stride;
  a.slot_stride = cache->slot_stride;
  a.head_stride = cache->head_stride;
  a.slot_count = cache->pages * cache->page_size;
  a.page = (uint32_t)cache->page_size;
  return rope_launch(a, dtype, T, cache->head_dim, rot_dim, interleaved, heads, (hipStream_t)stream);
}
