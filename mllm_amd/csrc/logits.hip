// Penalties for tokens that a row has seen, biases, and the tokens that a grammar allows, on logits, for gfx950.
//
//   seen in the row's history:            x = x > 0 ? x / r : x * r
//   n times among the generated ones:     x = x - (frequency * n + presence)
//   a bias for the token:                 x = x + bias
//   its bit in the row's mask is 0:       x = -inf
//
// A workgroup has a slice of a row: it counts in LDS which of the history's tokens fall into the slice, then goes over the slice's logits once.  Counts are
// integers and of several biases for a token the last one counts (the largest index, by a maximum), so nothing depends on the order of the atomics.
//
// What bounds it: one row, a launch (kernel 4.4 us) and the call.  96 bf16 rows of 151 936 with histories of up to 6000 tokens 23.6 us (61 MB: 2.6 TB/s; a copy of 2 GB has 5.18): the
// histories, which each of the 38 slices of a row goes through, on all eight XCDs; without them 62 rows of 233 096 14.0 us (4.1 TB/s).
#include "item8.h"

namespace mllmhip {

struct LogitsArgs {
  const void* x;
  void* y;
  int64_t x_row, y_row;
  int V;
  const int32_t *history, *length, *prompt;
  int64_t history_row;
  int history_len;
  const float *repetition, *presence, *frequency;
  const int32_t* bias_token;
  const float* bias;
  int64_t bias_token_row, bias_row;
  int biases;
  const uint32_t* masks;
  int64_t mask_row;
  int64_t nmasks;
  const int32_t* mask_of;
};

static constexpr uint32_t LOG_PROMPT = 1u << 31;  // beside a token's count: it is among the given ones

template <int XT>
__device__ __forceinline__ float element(const void* p, int64_t i) {
  return XT == MLLM_HIP_F32 ? reinterpret_cast<const float*>(p)[i] : bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}
// eight numbers that came from such a tensor, as they lie in it
template <int XT>
__device__ __forceinline__ void item_of(const float (&v)[8], Item8<XT>& it) {
  if constexpr (XT == MLLM_HIP_F32) {
    it.r[0] = u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    it.r[1] = u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
  } else {
    auto pair = [](float lo, float hi) { return __float_as_uint(lo) >> 16 | (__float_as_uint(hi) & 0xffff0000u); };
    it.r[0] = u32x4{pair(v[0], v[1]), pair(v[2], v[3]), pair(v[4], v[5]), pair(v[6], v[7])};
  }
}
template <int XT>
__device__ __forceinline__ void put_element(void* p, int64_t i, float v) {
  if (XT == MLLM_HIP_F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
}

// SLICE elements by WG threads, eight at a time each: what a slice reads is asked for in front of the counting.
template <int XT, int SLICE, int WG, bool BIASED>
__global__ __launch_bounds__(WG) void logits_kernel(LogitsArgs a) {
  constexpr int N = SLICE / WG / 8, AHEAD = 8;
  __shared__ __align__(16) uint32_t s_count[SLICE];
  __shared__ __align__(16) int s_bias[BIASED ? SLICE : 4];
  const int tid = threadIdx.x, row = blockIdx.y;
  const char* x = reinterpret_cast<const char*>(a.x) + row * a.x_row * (XT == MLLM_HIP_F32 ? 4 : 2);
  char* y = reinterpret_cast<char*>(a.y) + row * a.y_row * (XT == MLLM_HIP_F32 ? 4 : 2);
  // Items of eight elements begin where x is 16-byte aligned: in front of the row's first element where that is not.
  const int shift = (int)(reinterpret_cast<uintptr_t>(x) % 16) / (XT == MLLM_HIP_F32 ? 4 : 2);
  const bool same = reinterpret_cast<uintptr_t>(y) % 16 == reinterpret_cast<uintptr_t>(x) % 16;
  const int lo = (int)blockIdx.x * SLICE - shift, hi = min(lo + SLICE, a.V), real = max(lo, 0);
  const int said = a.history ? min(max(a.length ? a.length[row] : a.history_len, 0), a.history_len) : 0;
  const int given = a.prompt ? a.prompt[row] : 0;
  const float r = a.repetition ? a.repetition[row] : 1.0f, presence = a.presence ? a.presence[row] : 0.0f, frequency = a.frequency ? a.frequency[row] : 0.0f;
  const int64_t m = a.masks ? (a.mask_of ? (int64_t)a.mask_of[row] : row) : -1;
  const uint32_t* mask = m >= 0 && m < a.nmasks ? a.masks + m * a.mask_row : nullptr;
  const int words = (a.V + 31) / 32;
  const int32_t* h = a.history + row * a.history_row;
  int ahead[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; j++) ahead[j] = j * WG + tid < said ? h[j * WG + tid] : -1;
  Item8<XT> it[N];
  uint32_t low[N], high[N];  // words of the mask that eight bits from the first on lie in
#pragma unroll
  for (int n = 0; n < N; n++) {
    const int e = lo + (n * WG + tid) * 8, from = max(e, 0);
    it[n] = Item8<XT>{};
    if (e >= 0 && e + 8 <= a.V) {
      item_load<XT>(x, e, it[n]);
    } else if (e < a.V) {  // one of a row's ends
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = e + j >= 0 && e + j < a.V ? element<XT>(x, e + j) : 0.f;
      item_of<XT>(v, it[n]);
    }
    low[n] = high[n] = ~0u;
    if (mask && from < a.V) {
      low[n] = mask[from >> 5];
      if ((from >> 5) + 1 < words) high[n] = mask[(from >> 5) + 1];
    }
  }
  const bool counts = said > 0;
  if (counts || BIASED) {
#pragma unroll
    for (int i = tid * 4; i < SLICE; i += WG * 4) {
      *reinterpret_cast<u32x4*>(s_count + i) = u32x4{0, 0, 0, 0};
      if (BIASED) *reinterpret_cast<u32x4*>(s_bias + i) = u32x4{0, 0, 0, 0};
    }
    __syncthreads();
    for (int i0 = 0; i0 < said; i0 += AHEAD * WG) {
      int token[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; j++) {
        token[j] = ahead[j];
        const int next = i0 + (AHEAD + j) * WG + tid;
        ahead[j] = next < said ? h[next] : -1;
      }
#pragma unroll
      for (int j = 0; j < AHEAD; j++) {
        const int t = token[j], i = i0 + j * WG + tid;
        if (t < real || t >= hi) continue;
        if (i < given) atomicOr(&s_count[t - lo], LOG_PROMPT);
        else atomicAdd(&s_count[t - lo], 1u);
      }
    }
    if (BIASED) {
      const int32_t* bt = a.bias_token + row * a.bias_token_row;
      for (int i = tid; i < a.biases; i += WG) {
        const int t = bt[i];
        if (t >= real && t < hi) atomicMax(&s_bias[t - lo], i + 1);
      }
    }
    __syncthreads();
  }
  const float* bias = a.bias + row * a.bias_row;
#pragma unroll
  for (int n = 0; n < N; n++) {
    const int i = (n * WG + tid) * 8, e = lo + i;
    if (e >= a.V) break;
    float v[8];
    item_to_f32<XT>(it[n], v);
    // (bits in front of the row's first are of elements that are not there)
    const uint32_t allowed = (uint32_t)(((uint64_t)high[n] << 32 | low[n]) >> (max(e, 0) & 31)) << (max(e, 0) - e);
    if (counts) {
      const u32x4 c0 = *reinterpret_cast<const u32x4*>(s_count + i), c1 = *reinterpret_cast<const u32x4*>(s_count + i + 4);
      const uint32_t c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
      if (c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const uint32_t k = c[j] & ~LOG_PROMPT;
          if (c[j]) v[j] = v[j] > 0.f ? v[j] / r : v[j] * r;
          if (k) v[j] -= frequency * (float)k + presence;
        }
      }
    }
    if (BIASED) {
      const u32x4 b0 = *reinterpret_cast<const u32x4*>(s_bias + i), b1 = *reinterpret_cast<const u32x4*>(s_bias + i + 4);
      const uint32_t b[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
      if (b[0] | b[1] | b[2] | b[3] | b[4] | b[5] | b[6] | b[7]) {
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (b[j]) v[j] += bias[b[j] - 1];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = allowed >> j & 1 ? v[j] : -INFINITY;
    if (e >= 0 && e + 8 <= a.V && same) {
      item_store<XT>(y, e, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (e + j >= 0 && e + j < a.V) put_element<XT>(y, e + j, v[j]);
    }
  }
}

}  // namespace mllmhip

using namespace mllmhip;

MLLM_API int mllm_hip_logits_adjust(const mllm_hip_logits* l, int dtype, int64_t rows, int64_t vocab, void* stream) {
  if (!l || (dtype != MLLM_HIP_F32 && dtype != MLLM_HIP_BF16) || rows < 0 || vocab < 1) return MLLM_HIP_E_BADARG;
  if (l->history_len < 0 || l->biases < 0 || l->masks_count < 0) return MLLM_HIP_E_BADARG;
  if (vocab > (1 << 24) || rows > 65535 || l->history_len > 0x40000000 || l->biases > 0x40000000) return MLLM_HIP_E_SHAPE;  // (the kernel's places go past the last by some thousands)
  if (rows == 0) return 0;
  if (!l->x || !l->y || (l->history_len && !l->history) || (l->biases && (!l->bias_tokens || !l->bias)) || (l->masks_count && !l->masks)) return MLLM_HIP_E_BADARG;
  if (l->masks_count && !l->mask_of && l->masks_count < rows) return MLLM_HIP_E_BADARG;
  if (l->x == l->y ? l->x_stride != l->y_stride && rows > 1 : false) return MLLM_HIP_E_BADARG;
  if (rows > 1 && (l->y_stride < 0 ? -l->y_stride : l->y_stride) < vocab) return MLLM_HIP_E_BADARG;
  const uintptr_t wide = dtype == MLLM_HIP_F32 ? 4 : 2;
  auto al = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (!al(l->x, wide) || !al(l->y, wide) || !al(l->history, 4) || !al(l->lengths, 4) || !al(l->prompts, 4) || !al(l->repetition, 4) || !al(l->presence, 4) || !al(l->frequency, 4) ||
      !al(l->bias_tokens, 4) || !al(l->bias, 4) || !al(l->masks, 4) || !al(l->mask_of, 4))
    return MLLM_HIP_E_ALIGN;
  LogitsArgs a = {};
  a.x = l->x;
  a.y = l->y;
  a.x_row = l->x_stride;
  a.y_row = l->y_stride;
  a.V = (int)vocab;
  a.history = l->history_len ? l->history : nullptr;
  a.history_row = l->history_stride;
  a.history_len = (int)l->history_len;
  a.length = l->lengths;
  a.prompt = l->prompts;
  a.repetition = l->repetition;
  a.presence = l->presence;
  a.frequency = l->frequency;
  a.bias_token = l->bias_tokens;
  a.bias = l->bias;
  a.bias_token_row = l->bias_tokens_stride;
  a.bias_row = l->bias_stride;
  a.biases = (int)l->biases;
  a.masks = l->masks_count ? l->masks : nullptr;
  a.mask_row = l->masks_stride;
  a.nmasks = l->masks_count;
  a.mask_of = l->mask_of;
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto kern, int slice, int threads) {
    hipLaunchKernelGGL(kern, dim3((unsigned)((vocab + 7 + slice - 1) / slice), (unsigned)rows), dim3(threads), 0, st, a);  // (up to seven elements that are not there in front)
  };
#define LOGITS(XT_, SLICE_, WG_)                                              \
  if (a.biases) go(logits_kernel<XT_, SLICE_, WG_, true>, SLICE_, WG_);       \
  else go(logits_kernel<XT_, SLICE_, WG_, false>, SLICE_, WG_)
#define LOGITS_T(XT_)                                   \
  if (small) { LOGITS(XT_, 2048, 256); }                \
  else if (far) { LOGITS(XT_, 8192, 512); }             \
  else { LOGITS(XT_, 4096, 512); }
  // Slices of 2048 while they all run at once (one fp32 row of 151 936, a history of 900: the kernel 4.4 us, in slices of 4096 6.7).  Every slice reads the row's history: long ones in
  // slices of 8192.  In slices of 4096 / 8192, 96 bf16 rows with 6000 tokens 23.6 / 25.7 us, 128 with 16 000 38.0 / 31.0, 64 fp32 rows with 2000 17.8 / 20.5.
  const bool small = rows * vocab <= 1024 * 2048, far = a.history && a.history_len > 8192;
  if (dtype == MLLM_HIP_F32) { LOGITS_T(MLLM_HIP_F32) }
  else { LOGITS_T(MLLM_HIP_BF16) }
#undef LOGITS_T
#undef LOGITS
  return (int)hipGetLastError();
}
