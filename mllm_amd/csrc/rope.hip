// RMSNorm of every query and key head and their rotation by position, and the same on the way into a paged cache, for gfx950.
//
//   n = x * (w * rms),  rms = 1 / sqrt(mean over the head (x^2) + epsilon)      (as mllm_hip_rmsnorm; left out without a weight)
//   pair (a, b) number j of a head at position p:  a' = a cos - b sin,  b' = b cos + a sin,  angle = p * inv_freq[j]
//   with positions on several axes (time, height, width): p is the token's position on axis axes[j]
//
// Everything is fp32 between the load and the one rounding of the store.  The angle is not: fp32 holds p * f of a far position to
// a tenth of a radian at best, so it is multiplied in fp64, reduced to a fraction of a turn there, and only that goes to fp32.
// A workgroup has one token: its cosines and sines are computed once into LDS (64 pairs of 128 wide heads) while the first heads
// are on their way from memory, and every head of the token uses them.  Per byte there is nothing else to do: bound by memory
// with many tokens, by the launch and two dependent loads with few.  32 query and 8 key heads of 128, norm and halves turned:
// 8191 bf16 tokens 43 us (168 MB: 3.9 TB/s, a copy of 2 GB has 4.96), one fp32 token 3.2 in the kernel; 6007 bf16 tokens of 16 query and 4 key heads,
// pairs turned, keys and values into the cache, 16.6 us (74 MB: 4.5 TB/s).  Several axes cost a lookup of the pair's axis and up to four positions per workgroup, loaded together: 5185 bf16 tokens of
// 32 query and 8 key heads of 128 on three axes 29.6 us (106 MB: 3.6 TB/s), four fp32 tokens into the cache 3.9 in the kernel.  Vector instructions are not hidden behind memory there: eight choices more an item
// take 10 %.
#include "item8.h"

namespace mllmhip {

enum { ROPE_OUT = 0, ROPE_KEYS = 1, ROPE_VALUES = 2 };  // where a part's heads go: a tensor, the cache's keys, the cache's values
struct RopeGroup {
  const void* x;
  void* y;
  const float* w;
  int64_t x_token, x_head, y_token, y_head;
  int heads, unit0, kind;  // unit0: the part's first unit of as many heads as a wave has at a time
};
struct RopeArgs {
  RopeGroup part[4];
  int nparts, units, D, rot, passes, add_unit_offset;
  float eps, inv_d;
  const int32_t* positions;
  const double* inv_freq;
  // positions of several axes: which one each pair turns by (null: there is one), elements from a token to the next, from an axis to the next
  const int32_t* axes;
  int64_t pos_token, pos_axis;
  int naxes;
  // the cache's addressing
  const int64_t* slots;
  int64_t page_stride, slot_stride, head_stride, slot_count;
  uint32_t page;
};

// The value of the lane L away on the other side of a group of 2 L (L a power of two): lane ^ L
template <int L>
__device__ __forceinline__ float across(float v) {
  if (L == 1) return dpp_f<0xB1>(v);                 // quad_perm [1,0,3,2]
  if (L == 2) return dpp_f<0x4E>(v);                 // quad_perm [2,3,0,1]
  if (L == 4) return dpp_f<0x1B>(dpp_f<0x141>(v));   // mirrored in eight, then in four
  if (L == 8) return dpp_f<0x128>(v);                // turned by eight of sixteen
  const u32x2 r = L == 16 ? lanes16(__float_as_uint(v)) : lanes32(__float_as_uint(v));
  const int lane = threadIdx.x & 63;
  return __uint_as_float(lane & L ? r.x : r.y);
}

// AXES: positions of several axes (a form of its own: with both in one, calls with one axis take 5 % longer.  8191 bf16 tokens of 32 query and 8 key heads of 128 45.7 / 43.3 us, one fp32 token 3.1 / 2.95).
// G lanes per head of up to 8 * G elements.  A wave has 64 / G heads of one part at a time -- addresses are numbers of the scalar unit -- and goes through
// `passes` of them, up to ROPE_AHEAD on their way from memory at once.
enum { ROPE_AHEAD = 3, ROPE_AXES = 4 };
template <int XT, int G, bool NEXT, bool AXES>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  __shared__ __align__(16) float s_cos[256];
  __shared__ __align__(16) float s_sin[256];
  __shared__ __align__(16) uint32_t s_other[AXES ? 256 : 4];  // 0 for a pair on no axis, whose elements do not look at one another (0 times infinity is no number), else ~0
  constexpr int H = 64 / G;
  const int tid = threadIdx.x, lane = tid & 63, lg = lane % G, e = lg * 8;
  const int64_t t = blockIdx.x;
  const int half = a.rot / 2;
  const int unit0 = (blockIdx.y * a.passes) * 4 + __builtin_amdgcn_readfirstlane(tid >> 6);  // of H heads
  struct Part {
    RopeGroup g;
    int head;  // this lane's, of the part
    bool live;
  };
  auto part_of = [&](int unit) {
    Part p;
    p.g = a.part[0];
#pragma unroll
    for (int j = 1; j < 4; j++)
      if (j < a.nparts && unit >= a.part[j].unit0) p.g = a.part[j];
    p.head = (unit - p.g.unit0) * H + lane / G;
    p.live = unit < a.units && p.head < p.g.heads && e < a.D;
    return p;
  };
  int64_t stored = -1;  // where the token's slot is in the cache
  if (a.slots) {
    const int64_t slot = a.slots[t];
    if (slot >= 0 && slot < a.slot_count) {
      const uint32_t page = (uint32_t)slot / a.page;
      stored = page * a.page_stride + ((uint32_t)slot - page * a.page) * a.slot_stride;
    }
  }
  for (int p0 = 0; p0 < a.passes; p0 += ROPE_AHEAD) {
    Item8<XT> it[ROPE_AHEAD] = {};
#pragma unroll
    for (int p = 0; p < ROPE_AHEAD; p++) {
      if (p0 + p >= a.passes) break;
      const Part q = part_of(unit0 + (p0 + p) * 4);
      if (q.live) item_load<XT>(q.g.x, t * q.g.x_token + q.head * q.g.x_head + e, it[p]);
    }
    if (p0 == 0 && half > 0) {
      if (tid < half) {
        int place = 0;
        bool on = true;
        if (AXES) {
          // The token's positions are numbers of the scalar unit, asked for beside the pair's axis: with an address from it they would come one trip to memory later.
          const int32_t* at = a.positions + t * a.pos_token;
          const uint32_t axis = (uint32_t)a.axes[tid];
#pragma unroll
          for (int i = 0; i < ROPE_AXES; i++) {
            const int there = i < a.naxes ? at[i * a.pos_axis] : 0;
            place = axis == (uint32_t)i ? there : place;
          }
          on = axis < (uint32_t)a.naxes;
          s_other[tid] = on ? ~0u : 0;
        } else {
          place = a.positions[t];
        }
        // turns in fp64: p * f is off by 2^-53 of itself, which at 2^20 radians is 1e-10
        double turn = (double)place * a.inv_freq[tid] * 0.15915494309189533577;
        turn -= rint(turn);
        if (!on) turn = 0;  // (whatever its frequency is)
        float sn, cs;
        sincospif(2.0f * (float)turn, &sn, &cs);
        s_cos[tid] = cs;
        s_sin[tid] = sn;
      }
      __syncthreads();
    }
#pragma unroll
    for (int p = 0; p < ROPE_AHEAD; p++) {
      if (p0 + p >= a.passes) return;
      const Part q = part_of(unit0 + (p0 + p) * 4);
      float v[8];
      item_to_f32<XT>(it[p], v);
      if (q.g.w) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) ss = fmaf(v[j], v[j], ss);
        ss = group_sum<G>(ss);
        // 1 / sqrt by the hardware's (off by an ulp) and a step of Newton's: within an ulp, in a fifth of the instructions of a division and a root
        const float m = fmaf(ss, a.inv_d, a.eps);
        auto root = [](float x) {
          const float r = __builtin_amdgcn_rsqf(x);
          return fmaf(r * 0.5f, fmaf(-x * r, r, 1.0f), r);
        };
        const bool normal = __builtin_amdgcn_classf(m, 1 << 8);
        float rms = normal ? root(m) : __builtin_amdgcn_rsqf(m);
        if (__builtin_expect(__ballot(!normal) != 0, 0)) rms = m > 0.f && m < 0x1p-126f ? root(m * 0x1p64f) * 0x1p32f : rms;  // (the hardware's takes what is subnormal for 0)
        if (q.live) {
          const float4 w0 = *reinterpret_cast<const float4*>(q.g.w + e), w1 = *reinterpret_cast<const float4*>(q.g.w + e + 4);
          const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
          for (int j = 0; j < 8; j++) v[j] = v[j] * ((a.add_unit_offset ? w[j] + 1.0f : w[j]) * rms);
        }
      }
      if (half > 0 && q.g.kind != ROPE_VALUES) {
        const bool turns = q.live && e < a.rot;
        if (NEXT) {
          if (turns) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float cs = s_cos[e / 2 + j], sn = s_sin[e / 2 + j], x = v[2 * j], y = v[2 * j + 1];
              const uint32_t other = AXES ? s_other[e / 2 + j] : ~0u;
              v[2 * j] = x * cs - __uint_as_float(__float_as_uint(y) & other) * sn;
              v[2 * j + 1] = y * cs + __uint_as_float(__float_as_uint(x) & other) * sn;
            }
          }
        } else {  // the other element of every pair is half / 8 lanes away
          const bool first = e < half;
          const int j0 = first ? e : e - half;
          float o[8], w[8];  // (masked in front of the exchange: behind it the kernel takes 2 % longer, with a choice between results 10 %)
#pragma unroll
          for (int j = 0; j < 8; j++) w[j] = v[j];
          if (AXES) {
            const uint32_t* at = s_other + min(j0, 248);  // (of lanes behind the pairs: any, looked at by none)
            const u32x4 m0 = *reinterpret_cast<const u32x4*>(at), m1 = *reinterpret_cast<const u32x4*>(at + 4);
            const uint32_t m[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = __uint_as_float(__float_as_uint(v[j]) & m[j]);
          }
          if (half == 8 * (G / 2)) {  // (the whole of a head of 8 G elements: the usual one)
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = across<G / 2>(w[j]);
          } else {
            const int from = first ? lane + half / 8 : lane - half / 8;
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = __shfl(w[j], from);
          }
          if (turns) {
            const float4 c0 = *reinterpret_cast<const float4*>(s_cos + j0), c1 = *reinterpret_cast<const float4*>(s_cos + j0 + 4);
            const float4 n0 = *reinterpret_cast<const float4*>(s_sin + j0), n1 = *reinterpret_cast<const float4*>(s_sin + j0 + 4);
            const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, sn[8] = {n0.x, n0.y, n0.z, n0.w, n1.x, n1.y, n1.z, n1.w};
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = first ? v[j] * cs[j] - o[j] * sn[j] : v[j] * cs[j] + o[j] * sn[j];
          }
        }
      }
      if (!q.live) continue;
      if (q.g.kind == ROPE_OUT) item_store<XT>(q.g.y, t * q.g.y_token + q.head * q.g.y_head + e, v);
      else if (stored >= 0) item_store<MLLM_HIP_BF16>(q.g.y, stored + q.head * a.head_stride + e, v);
    }
  }
}

static bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// a part as the kernel takes it: checks of the strides that 16-byte loads and stores need
static int rope_group(const mllm_hip_heads& p, int dtype, int64_t T, bool stored, RopeGroup& g) {
  const int wide = dtype == MLLM_HIP_F32 ? 4 : 2;
  if (!p.x || (stored && !p.y) || p.heads < 1) return MLLM_HIP_E_BADARG;
  if (p.heads > 65536) return MLLM_HIP_E_SHAPE;
  auto whole = [&](int64_t stride) { return stride * wide % 16 == 0; };
  if (!al16(p.x) || !whole(p.x_token_stride) || !whole(p.x_head_stride) || (p.weight && !al16(p.weight))) return MLLM_HIP_E_ALIGN;
  if (stored && (!al16(p.y) || !whole(p.y_token_stride) || !whole(p.y_head_stride))) return MLLM_HIP_E_ALIGN;
  if (stored && !own_places(p, T)) return MLLM_HIP_E_BADARG;
  g = RopeGroup{p.x, p.y, p.weight, p.x_token_stride, p.x_head_stride, p.y_token_stride, p.y_head_stride, p.heads, 0, ROPE_OUT};
  return 0;
}

// Workgroups of a token: one for all of its heads while there are tokens to fill the chip, else one per four units.
static const int64_t ROPE_FULL = 2048;

static int rope_launch(RopeArgs& a, int dtype, int64_t T, int head_dim, int rot_dim, int interleaved, hipStream_t st) {
  const int lanes = head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : head_dim <= 256 ? 32 : 64, per = 64 / lanes;
  a.units = 0;
  for (int i = 0; i < a.nparts; i++) {
    a.part[i].unit0 = a.units;
    a.units += (a.part[i].heads + per - 1) / per;
  }
  const int all = (a.units + 3) / 4;
  a.D = head_dim;
  a.inv_d = 1.0f / (float)head_dim;
  a.rot = rot_dim;
  a.passes = T * all <= ROPE_FULL ? 1 : all;
  const dim3 grid((unsigned)T, (unsigned)((all + a.passes - 1) / a.passes));
#define ROPE(XT_, G_)                                                                                                \
  if (a.axes) {                                                                                                      \
    if (interleaved) hipLaunchKernelGGL((rope_kernel<XT_, G_, true, true>), grid, dim3(256), 0, st, a);              \
    else hipLaunchKernelGGL((rope_kernel<XT_, G_, false, true>), grid, dim3(256), 0, st, a);                         \
  } else {                                                                                                           \
    if (interleaved) hipLaunchKernelGGL((rope_kernel<XT_, G_, true, false>), grid, dim3(256), 0, st, a);             \
    else hipLaunchKernelGGL((rope_kernel<XT_, G_, false, false>), grid, dim3(256), 0, st, a);                        \
  }
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

// positions of several axes
struct RopeAxes {
  int64_t axis_stride, token_stride;
  int n;
  const int32_t* axes;
};
static int rope_axes(RopeArgs& a, int64_t T, int rot_dim, const RopeAxes& x) {
  if (x.n < 1 || (T && rot_dim && !x.axes)) return MLLM_HIP_E_BADARG;
  if (x.n > ROPE_AXES) return MLLM_HIP_E_SHAPE;
  if (reinterpret_cast<uintptr_t>(x.axes) % 4) return MLLM_HIP_E_ALIGN;
  a.axes = x.axes;
  a.naxes = x.n;
  a.pos_axis = x.axis_stride;
  a.pos_token = x.token_stride;
  return 0;
}

// what both calls check of the rotation
static int rope_checks(int dtype, int64_t T, int head_dim, const int32_t* positions, const double* inv_freq, int rot_dim) {
  if ((dtype != MLLM_HIP_F32 && dtype != MLLM_HIP_BF16) || T < 0 || head_dim < 1 || rot_dim < 0) return MLLM_HIP_E_BADARG;
  if (T && rot_dim && (!positions || !inv_freq)) return MLLM_HIP_E_BADARG;
  if (head_dim % 8 || head_dim > 512 || rot_dim > head_dim || rot_dim % 16 || T > 0xffffff) return MLLM_HIP_E_SHAPE;
  if (reinterpret_cast<uintptr_t>(positions) % 4 || reinterpret_cast<uintptr_t>(inv_freq) % 8) return MLLM_HIP_E_ALIGN;
  return 0;
}

static int norm_rope(int nparts, const mllm_hip_heads* parts, int dtype, int64_t T, int head_dim, float epsilon, int add_unit_offset, const int32_t* positions,
                     const RopeAxes* axes, const double* inv_freq, int rot_dim, int interleaved, void* stream) {
  if (nparts < 1 || nparts > 4 || !parts) return MLLM_HIP_E_BADARG;
  RC_RET(rope_checks(dtype, T, head_dim, positions, inv_freq, rot_dim));
  RopeArgs a = {};
  if (axes) RC_RET(rope_axes(a, T, rot_dim, *axes));
  if (T == 0) return 0;  // (tensors without elements have no addresses)
  for (int i = 0; i < nparts; i++) RC_RET(rope_group(parts[i], dtype, T, true, a.part[i]));
  a.nparts = nparts;
  a.eps = epsilon;
  a.add_unit_offset = add_unit_offset;
  a.positions = positions;
  a.inv_freq = inv_freq;
  return rope_launch(a, dtype, T, head_dim, rot_dim, interleaved, (hipStream_t)stream);
}

static int append(const mllm_hip_heads* q, const mllm_hip_heads* k, const mllm_hip_heads* v, int dtype, int64_t T, const mllm_hip_kv_cache* cache, const int64_t* slots,
                  float epsilon, int add_unit_offset, const int32_t* positions, const RopeAxes* axes, const double* inv_freq, int rot_dim, int interleaved, void* stream) {
  if (!k || !v || !cache || !cache->k || !cache->v || (T && !slots) || cache->heads < 1 || cache->pages < 1 || cache->page_size < 1) return MLLM_HIP_E_BADARG;
  RC_RET(rope_checks(dtype, T, cache->head_dim, positions, inv_freq, rot_dim));
  if (k->heads != cache->heads || v->heads != cache->heads || cache->pages > 0x7fffffff / cache->page_size || cache->page_stride < 0 ||
      cache->slot_stride < 0 || cache->page_stride > 0x7fffffff || cache->slot_stride > 0x3fffffff / cache->page_size ||
      (cache->slot_stride == 0 && cache->page_size > 1))
    return MLLM_HIP_E_SHAPE;
  if (!al16(cache->k) || !al16(cache->v) || cache->page_stride % 8 || cache->slot_stride % 8 || cache->head_stride % 8 ||
      reinterpret_cast<uintptr_t>(slots) % 8)
    return MLLM_HIP_E_ALIGN;
  RopeArgs a = {};
  if (axes) RC_RET(rope_axes(a, T, rot_dim, *axes));
  if (T == 0) return 0;
  RC_RET(rope_group(*k, dtype, T, false, a.part[0]));
  RC_RET(rope_group(*v, dtype, T, false, a.part[1]));
  a.part[0].y = cache->k;
  a.part[0].kind = ROPE_KEYS;
  a.part[1].y = cache->v;
  a.part[1].kind = ROPE_VALUES;
  a.part[1].w = nullptr;
  a.nparts = 2;
  if (q) {
    RC_RET(rope_group(*q, dtype, T, true, a.part[2]));
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
  return rope_launch(a, dtype, T, cache->head_dim, rot_dim, interleaved, (hipStream_t)stream);
}

}  // namespace mllmhip

using namespace mllmhip;

MLLM_API int mllm_hip_qk_norm_rope(int nparts, const mllm_hip_heads* parts, int dtype, int64_t T, int head_dim, float epsilon,
                                   int add_unit_offset, const int32_t* positions, const double* inv_freq, int rot_dim,
                                   int interleaved, void* stream) {
  return norm_rope(nparts, parts, dtype, T, head_dim, epsilon, add_unit_offset, positions, nullptr, inv_freq, rot_dim, interleaved, stream);
}

MLLM_API int mllm_hip_qk_norm_rope_axes(int nparts, const mllm_hip_heads* parts, int dtype, int64_t T, int head_dim, float epsilon, int add_unit_offset,
                                        const int32_t* positions, int64_t axis_stride, int64_t token_stride, int naxes, const int32_t* axes,
                                        const double* inv_freq, int rot_dim, int interleaved, void* stream) {
  const RopeAxes x = {axis_stride, token_stride, naxes, axes};
  return norm_rope(nparts, parts, dtype, T, head_dim, epsilon, add_unit_offset, positions, &x, inv_freq, rot_dim, interleaved, stream);
}

MLLM_API int mllm_hip_kv_append(const mllm_hip_heads* q, const mllm_hip_heads* k, const mllm_hip_heads* v, int dtype, int64_t T,
                                const mllm_hip_kv_cache* cache, const int64_t* slots, float epsilon, int add_unit_offset,
                                const int32_t* positions, const double* inv_freq, int rot_dim, int interleaved, void* stream) {
  return append(q, k, v, dtype, T, cache, slots, epsilon, add_unit_offset, positions, nullptr, inv_freq, rot_dim, interleaved, stream);
}

MLLM_API int mllm_hip_kv_append_axes(const mllm_hip_heads* q, const mllm_hip_heads* k, const mllm_hip_heads* v, int dtype, int64_t T,
                                     const mllm_hip_kv_cache* cache, const int64_t* slots, float epsilon, int add_unit_offset, const int32_t* positions,
                                     int64_t axis_stride, int64_t token_stride, int naxes, const int32_t* axes, const double* inv_freq, int rot_dim,
                                     int interleaved, void* stream) {
  const RopeAxes x = {axis_stride, token_stride, naxes, axes};
  return append(q, k, v, dtype, T, cache, slots, epsilon, add_unit_offset, positions, &x, inv_freq, rot_dim, interleaved, stream);
}
