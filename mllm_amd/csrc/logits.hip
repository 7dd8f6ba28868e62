// Penalties for tokens that a row has seen, biases, and the tokens that a grammar allows, on logits, for gfx950.
//
//   seen in the row's history:            x = x > 0 ? x / r : x * r
//   n times among the generated ones:     x = x - (frequency * n + presence)
//   a bias for the token:                 x = x + bias
//   its bit in the row's mask is 0:       x = -inf
//
// A workgroup has a slice of a row: it counts in LDS which of the history's tokens fall into the slice, then goes over the slice's logits once.  Counts are
// integers and of several biases for a token the last one counts (the largest index, by a maximum), so nothing depends on the order of the atomics.
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

enum { LOG_SLICE = 4096, LOG_WG = 256 };
static constexpr uint32_t LOG_PROMPT = 1u << 31;  // beside a token's count: it is among the given ones

template <int XT>
__device__ __forceinline__ float element(const void* p, int64_t i) {
  return XT == MLLM_HIP_F32 ? reinterpret_cast<const float*>(p)[i] : bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}
template <int XT>
__device__ __forceinline__ void put_element(void* p, int64_t i, float v) {
  if (XT == MLLM_HIP_F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
}

template <int XT>
__global__ __launch_bounds__(LOG_WG) void logits_kernel(LogitsArgs a) {
  __shared__ __align__(16) uint32_t s_count[LOG_SLICE];
  __shared__ __align__(16) int s_bias[LOG_SLICE];
  const int tid = threadIdx.x, row = blockIdx.y;
  const char* x = reinterpret_cast<const char*>(a.x) + row * a.x_row * (XT == MLLM_HIP_F32 ? 4 : 2);
  char* y = reinterpret_cast<char*>(a.y) + row * a.y_row * (XT == MLLM_HIP_F32 ? 4 : 2);
  // Items of eight elements begin where x is 16-byte aligned: in front of the row's first element where that is not.
  const int shift = (int)(reinterpret_cast<uintptr_t>(x) % 16) / (XT == MLLM_HIP_F32 ? 4 : 2);
  const bool same = reinterpret_cast<uintptr_t>(y) % 16 == reinterpret_cast<uintptr_t>(x) % 16;
  const int lo = (int)blockIdx.x * LOG_SLICE - shift, hi = min(lo + LOG_SLICE, a.V);
  const int said = a.history ? min(max(a.length ? a.length[row] : a.history_len, 0), a.history_len) : 0;
  const int given = a.prompt ? a.prompt[row] : 0;
  const float r = a.repetition ? a.repetition[row] : 1.0f, presence = a.presence ? a.presence[row] : 0.0f, frequency = a.frequency ? a.frequency[row] : 0.0f;
  const bool counts = said > 0, biased = a.biases > 0;
  if (counts || biased) {
    for (int i = tid * 4; i < LOG_SLICE; i += LOG_WG * 4) {
      *reinterpret_cast<u32x4*>(s_count + i) = u32x4{0, 0, 0, 0};
      *reinterpret_cast<u32x4*>(s_bias + i) = u32x4{0, 0, 0, 0};
    }
    __syncthreads();
    const int32_t* h = a.history + row * a.history_row;
    for (int i = tid; i < said; i += LOG_WG) {
      const int t = h[i];
      if (t < max(lo, 0) || t >= hi) continue;
      if (i < given) atomicOr(&s_count[t - lo], LOG_PROMPT);
      else atomicAdd(&s_count[t - lo], 1u);
    }
    const int32_t* bt = a.bias_token + row * a.bias_token_row;
    for (int i = tid; i < a.biases; i += LOG_WG) {
      const int t = bt[i];
      if (t >= max(lo, 0) && t < hi) atomicMax(&s_bias[t - lo], i + 1);
    }
    __syncthreads();
  }
  const int64_t m = a.masks ? (a.mask_of ? (int64_t)a.mask_of[row] : row) : -1;
  const uint32_t* mask = m >= 0 && m < a.nmasks ? a.masks + m * a.mask_row : nullptr;
  const float* bias = a.bias + row * a.bias_row;
  const int words = (a.V + 31) / 32;
  for (int i = tid * 8; i < LOG_SLICE; i += LOG_WG * 8) {
    const int e = lo + i;
    if (e >= a.V) break;
    const bool whole = e >= 0 && e + 8 <= a.V;
    float v[8];
    if (whole) {
      Item8<XT> it;
      item_load<XT>(x, e, it);
      item_to_f32<XT>(it, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = e + j >= 0 && e + j < a.V ? element<XT>(x, e + j) : 0.f;
    }
    uint32_t allowed = 0xff;
    if (mask) {  // eight bits from bit e on (bits in front of the first are of elements that are not there)
      const int from = max(e, 0), w = from >> 5;
      uint64_t bits = mask[w];
      if (w + 1 < words) bits |= (uint64_t)mask[w + 1] << 32;
      allowed = (uint32_t)(bits >> (from & 31)) << (from - e);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (counts) {
        const uint32_t c = s_count[i + j], n = c & ~LOG_PROMPT;
        if (c) v[j] = v[j] > 0.f ? v[j] / r : v[j] * r;
        if (n) v[j] -= frequency * (float)n + presence;
      }
      if (biased) {
        const int at = s_bias[i + j];
        if (at) v[j] += bias[at - 1];
      }
      v[j] = allowed >> j & 1 ? v[j] : -INFINITY;
    }
    if (whole && same) {
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
  if (vocab > (1 << 24) || rows > 65535 || l->history_len > 0x7fffffff || l->biases > 0x7ffffffe) return MLLM_HIP_E_SHAPE;
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
  const dim3 grid((unsigned)((vocab + 7 + LOG_SLICE - 1) / LOG_SLICE), (unsigned)rows);  // (up to seven elements that are not there in front)
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MLLM_HIP_F32) hipLaunchKernelGGL((logits_kernel<MLLM_HIP_F32>), grid, dim3(LOG_WG), 0, st, a);
  else hipLaunchKernelGGL((logits_kernel<MLLM_HIP_BF16>), grid, dim3(LOG_WG), 0, st, a);
  return (int)hipGetLastError();
}
