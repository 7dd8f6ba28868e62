// Eviction from a paged cache by accumulated attention weights, for gfx950.
//
// Of every sequence's and key head's first `length` positions the first `first` and the last `recent` stay, of the others the ones with the largest weights (equal
// ones: lowest index first; a NaN is the smallest), `keep` in all.  They go, in their order, to the places 0 .. keep - 1 of the pages of another table: pages may be shared by sequences,
// so nothing is moved within them.
//
// Two launches.  The first finds for every head which positions stay: the smallest weight that does is found digit by digit (11, 11 and 10 bits of the weight's order
// in 32) by counting in LDS, and the positions are written in order by a count in front of each wave's share.  The second copies the rows.
//
// What bounds it: 2048 of 24 x 6000 positions, 8 heads of 128, 99 us: the copy 88 (403 MB: 4.6 TB/s), the first launch 12.  4096 of 16 384 positions of one sequence 22.5: the first launch 14.2, eight workgroups in a chain of
// three counts with three barriers each (16 masses a lane in registers: the call takes 33 with masses read again for every digit, as behind 16 384 positions), the copy 8.4.  16 384 of 65 536 104 us, 8192 of 32 768 55.
#include "item8.h"

namespace mllmhip {

struct EvictArgs {
  const float* mass;
  int64_t mass_seq, mass_head;
  const int32_t *table, *length, *to_table;
  int64_t table_stride, to_stride;
  int most;  // positions that a sequence can have
  int heads, keep, first, recent, D;
  uint16_t *k, *v;
  int64_t head_stride;
  uint32_t page_bytes, slot_bytes, pages, page, page_mul;  // key / page = (2 key * page_mul) >> 32 >> page_shift for key < 2^31
  int page_shift;
  int32_t* kept;
  float* kept_mass;
};

enum { EVICT_WG = 1024, EVICT_HELD = 16, EVICT_BINS = 2048 };

// larger weights, larger numbers; -0 as 0, a NaN below all numbers.  0 and ~0 are no weight's: a position that is not there, and one that stays whatever its weight.
__device__ __forceinline__ uint32_t weight_order(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return v != v ? 1 : b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Each wave has a run of the positions, 64 at a time a lane each.  HELD: up to EVICT_HELD of 64, whose order stays in registers; else it is worked out again every time.
template <bool HELD>
__device__ __forceinline__ void evict_select(const EvictArgs& a, const float* mass, int n, int32_t* kept, float* kept_mass) {
  __shared__ uint32_t s_bin[EVICT_BINS];
  __shared__ uint32_t s_wave[2][EVICT_WG / 64];
  __shared__ uint32_t s_found[2];
  constexpr int WAVES = EVICT_WG / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lo = a.first, hi = n - a.recent;  // the ones that go by their weights: more of them than `want`
  uint32_t want = a.keep - a.first - a.recent;
  const int share = (n + EVICT_WG - 1) / EVICT_WG, from = wave * share * 64 + lane;  // in 64s
  auto order_of = [&](int i, float w) { return i >= n ? 0u : i < lo || i >= hi ? ~0u : weight_order(w); };
  uint32_t k[HELD ? EVICT_HELD : 1];
  if constexpr (HELD) {
    float w[EVICT_HELD];
#pragma unroll
    for (int j = 0; j < EVICT_HELD; j++) w[j] = j < share && from + 64 * j < n ? mass[from + 64 * j] : 0.f;
    for (int i = tid; i < EVICT_BINS; i += EVICT_WG) s_bin[i] = 0;
#pragma unroll
    for (int j = 0; j < EVICT_HELD; j++) k[j] = j < share ? order_of(from + 64 * j, w[j]) : 0;
  } else {
    for (int i = tid; i < EVICT_BINS; i += EVICT_WG) s_bin[i] = 0;
  }
  // f(position, order) of every one of this lane's positions, the wave's 64 together
  auto each = [&](auto f) {
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < EVICT_HELD; j++)
        if (j < share) f(from + 64 * j, k[j]);
    } else {
      constexpr int U = 8;
      for (int j0 = 0; j0 < share; j0 += U) {
        float w[U];
#pragma unroll
        for (int j = 0; j < U; j++) w[j] = j0 + j < share && from + 64 * (j0 + j) < n ? mass[from + 64 * (j0 + j)] : 0.f;
#pragma unroll
        for (int j = 0; j < U; j++)
          if (j0 + j < share) f(from + 64 * (j0 + j), order_of(from + 64 * (j0 + j), w[j]));
      }
    }
  };
  // The want-th largest: `prefix` are its digits so far, `want` which one it is among those that begin with them.  (No weight begins with the eleven ones of ~0; positions that
  // are not there are below all.)
  uint32_t prefix = 0;
  const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
  __syncthreads();
  if (want == 0) {
    prefix = ~1u;  // between the ones that stay and all weights
  } else {
#pragma unroll
    for (int d = 0; d < 3; d++) {
      each([&](int, uint32_t x) {
        if (d == 0 ? x != 0 && x != ~0u : x >> (shifts[d] + bits[d]) == prefix) atomicAdd(&s_bin[x >> shifts[d] & ((1u << bits[d]) - 1)], 1u);
      });
      __syncthreads();
      // bins from the largest down, two a thread: the one that the want-th is in
      const int top = EVICT_BINS - 1 - 2 * tid;
      const uint32_t c0 = s_bin[top], c1 = s_bin[top - 1];
      uint32_t up = c0 + c1;
#pragma unroll
      for (int s = 1; s < 64; s <<= 1) {
        const uint32_t o = __shfl_up(up, s);
        up += lane >= s ? o : 0;
      }
      if (lane == 63) s_wave[0][wave] = up;
      s_bin[top] = s_bin[top - 1] = 0;  // (by the thread that has read them: for the next digit)
      __syncthreads();
      uint32_t front = up - c0 - c1;
#pragma unroll
      for (int w = 0; w < WAVES; w++) front += w < wave ? s_wave[0][w] : 0;
      if (front < want && want <= front + c0 + c1) {
        const bool first = want <= front + c0;
        s_found[0] = first ? top : top - 1;
        s_found[1] = want - front - (first ? 0 : c0);
      }
      __syncthreads();
      prefix = prefix << bits[d] | s_found[0];
      want = s_found[1];
    }
  }
  // of weights that equal the border the first `want` stay
  uint32_t above = 0, equal = 0;
  each([&](int, uint32_t x) {
    above += __popcll(__ballot(x > prefix));
    equal += __popcll(__ballot(x == prefix));
  });
  __syncthreads();
  if (lane == 0) {
    s_wave[0][wave] = above;
    s_wave[1][wave] = equal;
  }
  __syncthreads();
  above = equal = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) {
    above += w < wave ? s_wave[0][w] : 0;
    equal += w < wave ? s_wave[1][w] : 0;
  }
  const uint64_t below = (1ull << lane) - 1;
  each([&](int i, uint32_t x) {
    const uint64_t va = __ballot(x > prefix), ve = __ballot(x == prefix);
    const uint32_t e = equal + __popcll(ve & below);  // equal ones in front
    if (x > prefix || (x == prefix && e < want)) {
      const uint32_t at = above + __popcll(va & below) + min(e, want);
      kept[at] = i;
      kept_mass[at] = mass[i];
    }
    above += __popcll(va);
    equal += __popcll(ve);
  });
}

__global__ __launch_bounds__(EVICT_WG) void evict_select_kernel(EvictArgs a) {
  const int b = blockIdx.y, h = blockIdx.x, n = min(max(a.length[b], 0), a.most);
  const float* mass = a.mass + b * a.mass_seq + h * a.mass_head;
  int32_t* kept = a.kept + ((int64_t)b * a.heads + h) * a.keep;
  float* kept_mass = a.kept_mass + ((int64_t)b * a.heads + h) * a.keep;
  if (n <= a.keep) {
    for (int i = threadIdx.x; i < a.keep; i += EVICT_WG) {
      kept[i] = i < n ? i : -1;
      kept_mass[i] = i < n ? mass[i] : 0.f;
    }
  } else if (n <= EVICT_HELD * EVICT_WG) {
    evict_select<true>(a, mass, n, kept, kept_mass);
  } else {
    evict_select<false>(a, mass, n, kept, kept_mass);
  }
}

// Rows of keys and of values, 16 bytes a lane: lanes of a row take its pieces in turn.
template <int L>
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictArgs a) {
  constexpr int PER = 256 / L, U = 4;  // rows at a time; turns
  const int b = blockIdx.y / a.heads, h = blockIdx.y % a.heads, p0 = threadIdx.x % L, row = threadIdx.x / L;
  const int n = min(max(a.length[b], 0), a.most), m = min(n, a.keep);
  const int32_t* kept = a.kept + (int64_t)blockIdx.y * a.keep;
  const uint64_t k = (uint64_t)(uintptr_t)(a.k + h * a.head_stride), v_less_k = (uint64_t)(uintptr_t)a.v - (uint64_t)(uintptr_t)a.k;
  auto at = [&](const int32_t* table, int place, bool& good) {
    const uint32_t page = __umulhi(2 * (uint32_t)place, a.page_mul) >> a.page_shift, id = (uint32_t)table[page];
    good = id < a.pages;
    return k + (uint64_t)id * a.page_bytes + ((uint32_t)place - page * a.page) * a.slot_bytes;
  };
  const int32_t *from_table = a.table + b * a.table_stride, *to_table = a.to_table + b * a.to_stride;
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int place = (blockIdx.x * U + u) * PER + row;
    if (place >= m) return;
    bool good, stored;
    const uint64_t from = at(from_table, kept[place], good), to = at(to_table, place, stored);
    if (!stored) continue;
    for (int p = p0; p < a.D / 8; p += L) {
      u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
      if (good) {
        x = *reinterpret_cast<const __attribute__((address_space(1))) u32x4*>(from + p * 16);
        y = *reinterpret_cast<const __attribute__((address_space(1))) u32x4*>(from + v_less_k + p * 16);
      }
      *reinterpret_cast<__attribute__((address_space(1))) u32x4*>(to + p * 16) = x;
      *reinterpret_cast<__attribute__((address_space(1))) u32x4*>(to + v_less_k + p * 16) = y;
    }
  }
}

}  // namespace mllmhip

using namespace mllmhip;

MLLM_API int mllm_hip_kv_evict(const mllm_hip_kv_cache* cache, const float* mass, int64_t mass_stride, int64_t mass_head_stride, int64_t mass_len, const int32_t* block_table,
                               int64_t table_stride, int64_t table_len, const int32_t* lengths, int64_t B, const int32_t* to_table, int64_t to_stride, int64_t to_len, int64_t keep,
                               int64_t first, int64_t recent, int32_t* kept, float* kept_mass, void* stream) {
  if (!cache || !cache->k || !cache->v || cache->heads < 1 || cache->head_dim < 1 || cache->pages < 1 || cache->page_size < 1 || B < 0 || mass_len < 0 || table_len < 0 || to_len < 0 ||
      keep < 0 || first < 0 || recent < 0 || first > keep || recent > keep - first)
    return MLLM_HIP_E_BADARG;
  if (cache->head_dim % 8 || cache->head_dim > 512 || cache->heads > 65536 || cache->pages > 0x7fffffff / cache->page_size || cache->page_stride < 0 || cache->slot_stride < 0 ||
      cache->page_stride > 0x7fffffff || cache->slot_stride > 0x3fffffff / cache->page_size || (cache->slot_stride == 0 && cache->page_size > 1) ||
      table_len > 0x40000000 / cache->page_size || to_len > 0x40000000 / cache->page_size || B > 65535 / cache->heads || keep > to_len * cache->page_size)
    return MLLM_HIP_E_SHAPE;
  if (B == 0 || keep == 0) return 0;
  if ((mass_len && !mass) || (table_len && !block_table) || !lengths || !to_table || !kept || !kept_mass || kept_mass == mass) return MLLM_HIP_E_BADARG;
  auto al = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (!al(cache->k, 16) || !al(cache->v, 16) || cache->page_stride % 8 || cache->slot_stride % 8 || cache->head_stride % 8 || !al(mass, 4) || !al(block_table, 4) || !al(lengths, 4) ||
      !al(to_table, 4) || !al(kept, 4) || !al(kept_mass, 4))
    return MLLM_HIP_E_ALIGN;
  EvictArgs a = {};
  a.mass = mass;
  a.mass_seq = mass_stride;
  a.mass_head = mass_head_stride;
  a.table = block_table;
  a.table_stride = table_stride;
  a.length = lengths;
  a.to_table = to_table;
  a.to_stride = to_stride;
  const int64_t places = table_len * cache->page_size;
  a.most = (int)(mass_len < places ? mass_len : places);
  a.heads = cache->heads;
  a.keep = (int)keep;
  a.first = (int)first;
  a.recent = (int)recent;
  a.D = cache->head_dim;
  a.k = reinterpret_cast<uint16_t*>(cache->k);
  a.v = reinterpret_cast<uint16_t*>(cache->v);
  a.head_stride = cache->head_stride;
  a.page_bytes = (uint32_t)(cache->page_stride * 2);
  a.slot_bytes = (uint32_t)(cache->slot_stride * 2);
  a.pages = (uint32_t)cache->pages;
  a.page = (uint32_t)cache->page_size;
  int s = 0;
  while ((1ll << s) < cache->page_size) s++;
  a.page_mul = (uint32_t)(((1ull << (31 + s)) + cache->page_size - 1) / cache->page_size);
  a.page_shift = s;
  a.kept = kept;
  a.kept_mass = kept_mass;
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)cache->heads, (unsigned)B), dim3(EVICT_WG), 0, st, a);
  RC_RET((int)hipGetLastError());
  const int pieces = cache->head_dim / 8, lanes = pieces <= 8 ? 8 : pieces <= 16 ? 16 : 32, rows = 256 / lanes * 4;
  const dim3 grid((unsigned)((keep + rows - 1) / rows), (unsigned)(B * cache->heads));
  if (lanes == 8) hipLaunchKernelGGL(evict_copy_kernel<8>, grid, dim3(256), 0, st, a);
  else if (lanes == 16) hipLaunchKernelGGL(evict_copy_kernel<16>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(evict_copy_kernel<32>, grid, dim3(256), 0, st, a);
  return (int)hipGetLastError();
}
