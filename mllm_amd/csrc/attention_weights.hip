// What every key of a paged cache gets of the new tokens' attention, for gfx950.
//
//   mass_j = (j before the new tokens ? decay * mass_j : 0) + sum over rows r that see j of exp(s_rj - m_r) / l_r,   s_rj = scale * (q_r . k_j),
//   m_r = max_j s_rj,  l_r = sum_j exp(s_rj - m_r);  a row is a new token and a query head of the group that shares the key head.
//
// S^T = K Q^T on v_mfma_f32_16x16x32_bf16, as in the attention: the first operand is 16 keys, which a lane takes as 16-byte pieces of one key straight from the cache; a lane
// gets the scores of one row (lane % 16) with four keys.  Products of bf16 are exact, fp32 queries enter as three bf16 parts; scores, maxima and sums are fp32.
//
// A row's weights need its maximum and sum over all keys first, so there are two passes.
//   Up to 16 rows (a token): the first writes the scores, of 16 rows 64 bytes a key where a key of 128 has 256, with every wave's maxima and sums; the second joins
//   these and adds up the weights from the scores.  Keys are read once.
//   More rows: the first finds maxima and sums, a wave's rows in registers and keys going by (a small launch joins them where keys are cut into ranges); the second has a wave's
//   keys in registers and rows going by, so that what a key gets is a sum in a lane.
// No atomics: what a key gets is summed by one wave in one order.
#include "attention_common.h"

namespace mllmhip {

struct WeightArgs {
  const void* q;
  int64_t q_token, q_head;
  const uint16_t* k;
  int64_t head_stride;
  uint32_t page_bytes, slot_bytes, pages, page, page_mul;  // key / page = (2 key * page_mul) >> 32 >> page_shift for key < 2^31
  int page_shift;
  const int32_t* table;
  int64_t table_stride;
  int64_t places;  // that a sequence's row of the table has
  const int32_t *cu, *prefix;
  int T, B, kv, group, D, max_tokens, max_keys, ranges, row_tiles;
  float c, decay;  // scale * log2 e
  float* mass;
  int64_t mass_seq, mass_head, mass_len;
  // workspace
  float* score;  // [B][kv][rows][pitch]
  int rows, pitch;
  f32x2* ml;     // few rows: [range][B][kv][rows]; more: [range][T][heads], maximum (times c) and sum
  f32x2* row;    // [T][heads]: maximum (times c) and 1 / sum of all keys
};
__device__ u32x4 g_no_key[32];  // what a page outside the cache reads as (never written)

struct WeightSeq {
  int first, n, prefix, keys;  // its first row of q, numbers of new tokens, of positions before them and of positions that count
};
__device__ __forceinline__ WeightSeq weight_sequence(const WeightArgs& a, int b) {
  WeightSeq s;
  const int lo = max(a.cu[b], 0), hi = min(a.cu[b + 1], a.T);
  s.first = lo;
  s.n = max(hi - lo, 0);
  s.prefix = min(max(a.prefix[b], 0), (int)a.places);  // (positions behind the table are not there; sums of two such numbers are below 2^31)
  s.keys = min(min(s.prefix + s.n, (int)a.places), a.max_keys);
  s.n = min(s.n, a.max_tokens);
  return s;
}

// 16 bytes ks * 32 + 8 g .. of key `key` of a sequence
template <int KS>
__device__ __forceinline__ void load_key(const WeightArgs& a, const int32_t* table, uint64_t k_at, int key, bool there, int g, u32x4 (&r)[KS]) {
  const uint32_t page = __umulhi(2 * (uint32_t)key, a.page_mul) >> a.page_shift, id = (uint32_t)(there ? table[page] : -1);
  const bool good = id < a.pages;
  const uint64_t at = good ? k_at + (uint64_t)id * a.page_bytes + ((uint32_t)key - page * a.page) * a.slot_bytes : (uint64_t)(uintptr_t)g_no_key;
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    const int e = 32 * ks + 8 * g;
    r[ks] = *reinterpret_cast<const __attribute__((address_space(1))) u32x4*>(e < a.D ? at + e * 2 : (uint64_t)(uintptr_t)g_no_key);
  }
}

// Scores (times 1) of 16 keys and 16 rows.  With fp32 queries an infinite element of a key makes a NaN with the second and third part of a query's, which may be 0: it
// counts with the first alone, which has the sign.  Such scores, and those that are NaN anyway, are formed once more.
template <int KS, bool F32>
__device__ __forceinline__ at_f32x4 key_scores(const u32x4 (&k)[KS], const at_bf16x8 (&q)[KS][F32 ? 3 : 1]) {
  at_f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < KS; ks++)
#pragma unroll
    for (int p = (F32 ? 3 : 1) - 1; p >= 0; p--) s = mma(frag(k[ks]), q[ks][p], s);
  if constexpr (F32) {
    const float all = (s[0] + s[1]) + (s[2] + s[3]);
    if (__builtin_expect(__ballot(all != all) != 0, 0)) {
      s = at_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const at_bf16x8 f = frag(u32x4{finite_pair(k[ks].x), finite_pair(k[ks].y), finite_pair(k[ks].z), finite_pair(k[ks].w)});
        s = mma(f, q[ks][2], s);
        s = mma(f, q[ks][1], s);
        s = mma(frag(k[ks]), q[ks][0], s);
      }
    }
  }
  return s;
}
// Rows r0 .. r0 + 15 of a sequence as an operand: row `col` of lane col
template <int KS, bool F32>
__device__ __forceinline__ void load_rows(const WeightArgs& a, const WeightSeq& s, int h, int r, int rows, int g, at_bf16x8 (&q)[KS][F32 ? 3 : 1]) {
  const bool live = r < rows;
  const int token = live ? r / a.group : 0, head = h * a.group + (live ? r - token * a.group : 0);
  const int64_t at = (s.first + token) * a.q_token + head * a.q_head + 8 * g;
#pragma unroll
  for (int ks = 0; ks < KS; ks++) query_parts<F32>(a.q, at + 32 * ks, live && 32 * ks + 8 * g < a.D, q[ks]);
}
// a lane's maximum m (times c) and sum l with four more scores
__device__ __forceinline__ void take(float& m, float& l, const at_f32x4& s, float c) {
  const float top = larger(larger(s[0], s[1]), larger(s[2], s[3])) * c;
  const float next = larger(m, top), ref = next == -INFINITY ? 0.f : next;
  l *= __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
  for (int j = 0; j < 4; j++) l += __builtin_amdgcn_exp2f(fmaf(s[j], c, -ref));
  m = next;
}
__device__ __forceinline__ void join(float& m, float& l, float m2, float l2) {
  const float next = larger(m, m2), ref = next == -INFINITY ? 0.f : next;
  l = l * __builtin_amdgcn_exp2f(m - ref) + l2 * __builtin_amdgcn_exp2f(m2 - ref);
  m = next;
}
__device__ __forceinline__ void join_lanes(float& m, float& l) {  // over the four lanes of a row
#pragma unroll
  for (int d = 16; d <= 32; d *= 2) join(m, l, __shfl_xor(m, d), __shfl_xor(l, d));
}
// the number that a row's exponents are less, and what they are multiplied by: a row that sees nothing has no weights
__device__ __forceinline__ f32x2 final_row(float m, float l) { return f32x2{m == -INFINITY ? 0.f : m, l == 0.f ? 0.f : 1.0f / l}; }

// ---- up to 16 rows --------------------------------------------------------------------------------------------------------
template <int KS, bool F32>
__global__ __launch_bounds__(256) void weights_scores_kernel(WeightArgs a) {
  __shared__ f32x2 s_ml[4][16];
  const int h = blockIdx.y % a.kv, b = blockIdx.y / a.kv, range = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const WeightSeq s = weight_sequence(a, b);
  const int rows = min(s.n * a.group, a.rows);
  if (rows == 0) return;
  const int per = ((s.keys + a.ranges - 1) / a.ranges + 63) / 64 * 64, begin = range * per, end = min(begin + per, s.keys);
  const int32_t* table = a.table + b * a.table_stride;
  const uint64_t k_at = (uint64_t)(uintptr_t)(a.k + h * a.head_stride);
  at_bf16x8 q[KS][F32 ? 3 : 1];
  load_rows<KS, F32>(a, s, h, col, rows, g, q);
  const int token = col < rows ? col / a.group : -1;
  float m = -INFINITY, l = 0.f;
  float* score = a.score + ((int64_t)blockIdx.y * a.rows + col) * a.pitch;
  for (int k0 = begin + wave * 16; k0 < end; k0 += 64) {
    u32x4 k[KS];
    load_key<KS>(a, table, k_at, k0 + col, k0 + col < end, g, k);
    at_f32x4 y = key_scores<KS, F32>(k, q);
    const int seen = min(s.prefix + token + 1, end) - (k0 + 4 * g);  // of this lane's keys
#pragma unroll
    for (int j = 0; j < 4; j++) y[j] = j < seen && token >= 0 ? y[j] : -INFINITY;
    if (col < a.rows) *reinterpret_cast<at_f32x4*>(score + k0 + 4 * g) = y;
    take(m, l, y, a.c);
  }
  join_lanes(m, l);
  if (g == 0) s_ml[wave][col] = f32x2{m, l};
  __syncthreads();
  if (threadIdx.x < a.rows) {
    for (int w = 1; w < 4; w++) join(m, l, s_ml[w][col].x, s_ml[w][col].y);
    a.ml[((int64_t)range * gridDim.y + blockIdx.y) * a.rows + col] = f32x2{m, l};
  }
}

__global__ __launch_bounds__(256) void weights_sum_kernel(WeightArgs a) {
  __shared__ f32x2 s_row[16];
  const int h = blockIdx.y % a.kv, b = blockIdx.y / a.kv;
  const WeightSeq s = weight_sequence(a, b);
  if (s.n == 0) return;
  if (threadIdx.x < a.rows) {
    float m = -INFINITY, l = 0.f;
    for (int r = 0; r < a.ranges; r++) {
      const f32x2 x = a.ml[((int64_t)r * gridDim.y + blockIdx.y) * a.rows + threadIdx.x];
      join(m, l, x.x, x.y);
    }
    s_row[threadIdx.x] = final_row(m, l);
  }
  __syncthreads();
  const int key = blockIdx.x * 256 + threadIdx.x;
  if (key >= s.keys || key >= a.mass_len) return;
  const float* score = a.score + (int64_t)blockIdx.y * a.rows * a.pitch + key;
  float sum = 0.f;
  for (int r = 0; r < a.rows; r++) {
    const float p = __builtin_amdgcn_exp2f(fmaf(score[(int64_t)r * a.pitch], a.c, -s_row[r].x)) * s_row[r].y;
    sum += key <= s.prefix + r / a.group ? p : 0.f;  // (a row without a number has none for keys that it sees)
  }
  float* mass = a.mass + b * a.mass_seq + h * a.mass_head + key;
  *mass = key < s.prefix && a.decay != 0.f ? a.decay * *mass + sum : sum;
}

// ---- more rows ------------------------------------------------------------------------------------------------------------
enum { WEIGHT_NQ = 2, WEIGHT_ROWS = 4 * WEIGHT_NQ * 16, WEIGHT_NK = 2, WEIGHT_KEYS = 4 * WEIGHT_NK * 16 };

template <int KS, bool F32>
__global__ __launch_bounds__(256) void weights_max_kernel(WeightArgs a) {
  constexpr int NQ = WEIGHT_NQ;
  const int h = blockIdx.y % a.kv, b = blockIdx.y / a.kv, range = blockIdx.x % a.ranges, rt = blockIdx.x / a.ranges;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const WeightSeq s = weight_sequence(a, b);
  const int rows = s.n * a.group, row0 = rt * WEIGHT_ROWS + wave * NQ * 16;
  if (row0 >= rows) return;
  // (keys behind this wave's last token are seen by none of its rows)
  const int last = (min(rows, row0 + NQ * 16) - 1) / a.group;
  const int per = ((s.keys + a.ranges - 1) / a.ranges + 15) / 16 * 16, begin = range * per, end = min(min(begin + per, s.keys), s.prefix + last + 1);
  const int32_t* table = a.table + b * a.table_stride;
  const uint64_t k_at = (uint64_t)(uintptr_t)(a.k + h * a.head_stride);
  at_bf16x8 q[NQ][KS][F32 ? 3 : 1];
  int token[NQ];
  float m[NQ], l[NQ];
#pragma unroll
  for (int i = 0; i < NQ; i++) {
    const int r = row0 + i * 16 + col;
    load_rows<KS, F32>(a, s, h, r, rows, g, q[i]);
    token[i] = r < rows ? r / a.group : -1;
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  for (int k0 = begin; k0 < end; k0 += 16) {
    u32x4 k[KS];
    load_key<KS>(a, table, k_at, k0 + col, k0 + col < end, g, k);
#pragma unroll
    for (int i = 0; i < NQ; i++) {
      at_f32x4 y = key_scores<KS, F32>(k, q[i]);
      const int seen = min(s.prefix + token[i] + 1, end) - (k0 + 4 * g);
#pragma unroll
      for (int j = 0; j < 4; j++) y[j] = j < seen && token[i] >= 0 ? y[j] : -INFINITY;
      take(m[i], l[i], y, a.c);
    }
  }
  const int heads = a.kv * a.group;
#pragma unroll
  for (int i = 0; i < NQ; i++) {
    join_lanes(m[i], l[i]);
    if (g || token[i] < 0) continue;
    const int64_t at = (int64_t)(s.first + token[i]) * heads + h * a.group + (row0 + i * 16 + col - token[i] * a.group);
    if (a.ranges == 1) a.row[at] = final_row(m[i], l[i]);
    else a.ml[(int64_t)range * a.T * heads + at] = f32x2{m[i], l[i]};
  }
}

__global__ __launch_bounds__(256) void weights_join_kernel(WeightArgs a) {
  const int64_t all = (int64_t)a.T * a.kv * a.group, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  float m = -INFINITY, l = 0.f;
  for (int r = 0; r < a.ranges; r++) join(m, l, a.ml[r * all + i].x, a.ml[r * all + i].y);  // (rows of no sequence: any numbers, never used)
  a.row[i] = final_row(m, l);
}

template <int KS, bool F32>
__global__ __launch_bounds__(256) void weights_mass_kernel(WeightArgs a) {
  constexpr int NK = WEIGHT_NK;
  const int h = blockIdx.y % a.kv, b = blockIdx.y / a.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const WeightSeq s = weight_sequence(a, b);
  const int rows = s.n * a.group, k0 = blockIdx.x * WEIGHT_KEYS + wave * NK * 16;
  if (rows == 0 || k0 >= s.keys) return;
  const int32_t* table = a.table + b * a.table_stride;
  const uint64_t k_at = (uint64_t)(uintptr_t)(a.k + h * a.head_stride);
  u32x4 k[NK][KS];
  at_f32x4 sum[NK];
#pragma unroll
  for (int i = 0; i < NK; i++) {
    const int key = k0 + i * 16 + col;
    load_key<KS>(a, table, k_at, key, key < s.keys, g, k[i]);
    sum[i] = at_f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int heads = a.kv * a.group;
  const int from = max(k0 - s.prefix, 0) * a.group / 16 * 16;  // the first token that sees the first of these keys
  for (int r0 = from; r0 < rows; r0 += 16) {
    at_bf16x8 q[KS][F32 ? 3 : 1];
    const int r = r0 + col;
    load_rows<KS, F32>(a, s, h, r, rows, g, q);
    const int token = r < rows ? r / a.group : -1;
    const f32x2 row = token >= 0 ? a.row[(int64_t)(s.first + token) * heads + h * a.group + (r - token * a.group)] : f32x2{0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NK; i++) {
      at_f32x4 y = key_scores<KS, F32>(k[i], q);
      const int seen = min(s.prefix + token + 1, s.keys) - (k0 + i * 16 + 4 * g);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float p = __builtin_amdgcn_exp2f(fmaf(y[j], a.c, -row.x)) * row.y;
        sum[i][j] += j < seen && token >= 0 ? p : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NK; i++) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float v = group_sum<16>(sum[i][j]);
      const int key = k0 + i * 16 + 4 * g + j;
      if (col != j || key >= s.keys || key >= a.mass_len) continue;
      float* mass = a.mass + b * a.mass_seq + h * a.mass_head + key;
      *mass = key < s.prefix && a.decay != 0.f ? a.decay * *mass + v : v;
    }
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------
struct WeightPlan {
  bool few;
  int rows, pitch, ranges, row_tiles;
};
static WeightPlan weight_plan(int64_t B, int heads, int kv, int64_t max_tokens, int64_t max_keys) {
  WeightPlan p = {};
  const int64_t rows = max_tokens * (heads / kv);
  p.few = rows <= 16;
  p.rows = p.few ? (int)rows : 0;
  p.pitch = (int)((max_keys + 63) / 64 * 64);
  p.row_tiles = p.few ? 1 : (int)((rows + WEIGHT_ROWS - 1) / WEIGHT_ROWS);
  const int64_t uncut = B * kv * p.row_tiles, most = (max_keys + 255) / 256, wanted = (1023 + uncut) / uncut;
  p.ranges = (int)(uncut >= 1024 || most < 2 ? 1 : wanted < most ? wanted : most);
  return p;
}
static size_t weight_room(const WeightPlan& p, int64_t T, int64_t B, int heads, int kv) {
  if (p.few) return ((size_t)B * kv * p.rows * p.pitch + (size_t)p.ranges * B * kv * p.rows * 2) * sizeof(float);
  return (size_t)(p.ranges > 1 ? p.ranges + 1 : 1) * T * heads * 2 * sizeof(float);
}
static bool weight_sizes(int dtype, int64_t T, int64_t B, int heads, int kv, int head_dim, int64_t max_tokens, int64_t max_keys) {
  return (dtype == MLLM_HIP_F32 || dtype == MLLM_HIP_BF16) && T >= 0 && B >= 0 && heads >= 1 && kv >= 1 && head_dim >= 1 && max_tokens >= 0 && max_keys >= 0;
}
static bool weight_shape(int64_t T, int64_t B, int heads, int kv, int head_dim, int64_t max_tokens, int64_t max_keys) {
  return head_dim % 8 == 0 && head_dim <= 256 && heads % kv == 0 && heads <= 65536 && T <= 0x3fffffff / heads && B <= 65535 / kv && max_tokens <= 0x7fffffff / heads &&
         max_keys <= 0x40000000;
}

}  // namespace mllmhip

using namespace mllmhip;

MLLM_API size_t mllm_hip_attention_weights_workspace_bytes(int dtype, int64_t T, int64_t B, int heads, int kv_heads, int head_dim, int64_t max_tokens, int64_t max_keys) {
  if (!weight_sizes(dtype, T, B, heads, kv_heads, head_dim, max_tokens, max_keys) || !weight_shape(T, B, heads, kv_heads, head_dim, max_tokens, max_keys)) return 0;
  if (T == 0 || B == 0 || max_tokens == 0 || max_keys == 0) return 0;
  if (max_tokens > T) max_tokens = T;
  return weight_room(weight_plan(B, heads, kv_heads, max_tokens, max_keys), T, B, heads, kv_heads);
}

MLLM_API int mllm_hip_attention_weights(const mllm_hip_heads* q, int dtype, int64_t T, const mllm_hip_kv_cache* cache, float* mass, int64_t mass_stride,
                                        int64_t mass_head_stride, int64_t mass_len, const int32_t* block_table, int64_t table_stride, int64_t table_len,
                                        const int32_t* cu_tokens, const int32_t* prefix, int64_t B, int64_t max_tokens, int64_t max_keys, float decay, float scale,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !cache || table_len < 0 || mass_len < 0 || !(scale > 0.f) || scale > 2e38f || !(decay >= 0.f) || decay > 2e38f || cache->pages < 1 || cache->page_size < 1)
    return MLLM_HIP_E_BADARG;
  if (!weight_sizes(dtype, T, B, q->heads, cache->heads, cache->head_dim, max_tokens, max_keys)) return MLLM_HIP_E_BADARG;
  if (!weight_shape(T, B, q->heads, cache->heads, cache->head_dim, max_tokens, max_keys) || cache->pages > 0x7fffffff / cache->page_size ||
      table_len > 0x40000000 / cache->page_size || cache->page_stride < 0 || cache->slot_stride < 0 || cache->page_stride > 0x7fffffff ||
      cache->slot_stride > 0x3fffffff / cache->page_size || (cache->slot_stride == 0 && cache->page_size > 1))
    return MLLM_HIP_E_SHAPE;
  if (T == 0 || B == 0 || max_tokens == 0 || max_keys == 0) return 0;
  if (max_tokens > T) max_tokens = T;
  if (!q->x || !cache->k || !block_table || !cu_tokens || !prefix || table_len < 1 || (mass_len && !mass)) return MLLM_HIP_E_BADARG;
  if ((B > 1 && !mass_stride) || (cache->heads > 1 && !mass_head_stride)) return MLLM_HIP_E_BADARG;
  const int wide = dtype == MLLM_HIP_F32 ? 4 : 2;
  auto al = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (!al(q->x, 16) || !al(cache->k, 16) || q->x_token_stride * wide % 16 || q->x_head_stride * wide % 16 || cache->page_stride % 8 || cache->slot_stride % 8 ||
      cache->head_stride % 8 || !al(mass, 4) || !al(block_table, 4) || !al(cu_tokens, 4) || !al(prefix, 4) || !al(workspace, 16))
    return MLLM_HIP_E_ALIGN;
  const int heads = q->heads, D = cache->head_dim;
  const bool f32 = dtype == MLLM_HIP_F32;
  const WeightPlan p = weight_plan(B, heads, cache->heads, max_tokens, max_keys);
  const size_t need = weight_room(p, T, B, heads, cache->heads);
  if (!workspace || workspace_bytes < need) return MLLM_HIP_E_BADARG;
  if (p.row_tiles > 0xffffff / p.ranges) return MLLM_HIP_E_SHAPE;
  WeightArgs a = {};
  a.q = q->x;
  a.q_token = q->x_token_stride;
  a.q_head = q->x_head_stride;
  a.k = reinterpret_cast<const uint16_t*>(cache->k);
  a.head_stride = cache->head_stride;
  a.page_bytes = (uint32_t)(cache->page_stride * 2);
  a.slot_bytes = (uint32_t)(cache->slot_stride * 2);
  a.pages = (uint32_t)cache->pages;
  a.page = (uint32_t)cache->page_size;
  int s = 0;
  while ((1ll << s) < cache->page_size) s++;
  a.page_mul = (uint32_t)(((1ull << (31 + s)) + cache->page_size - 1) / cache->page_size);
  a.page_shift = s;
  a.table = block_table;
  a.table_stride = table_stride;
  a.places = table_len * cache->page_size;
  a.cu = cu_tokens;
  a.prefix = prefix;
  a.T = (int)T;
  a.B = (int)B;
  a.kv = cache->heads;
  a.group = heads / cache->heads;
  a.D = D;
  a.max_tokens = (int)max_tokens;
  a.max_keys = (int)max_keys;
  a.ranges = p.ranges;
  a.row_tiles = p.row_tiles;
  a.c = scale * 1.44269504088896341f;
  a.decay = decay;
  a.mass = mass;
  a.mass_seq = mass_stride;
  a.mass_head = mass_head_stride;
  a.mass_len = mass_len;
  a.rows = p.rows;
  a.pitch = p.pitch;
  hipStream_t st = (hipStream_t)stream;
  const unsigned heads_of_all = (unsigned)(B * cache->heads);
#define KSTEPS(KERNEL_, GRID_)                                                                                \
  {                                                                                                           \
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, GRID_, dim3(256), 0, st, a); };                       \
    if (D <= 64) { if (f32) go(KERNEL_<2, true>); else go(KERNEL_<2, false>); }                               \
    else if (D <= 96) { if (f32) go(KERNEL_<3, true>); else go(KERNEL_<3, false>); }                          \
    else if (D <= 128) { if (f32) go(KERNEL_<4, true>); else go(KERNEL_<4, false>); }                         \
    else { if (f32) go(KERNEL_<8, true>); else go(KERNEL_<8, false>); }                                       \
    RC_RET((int)hipGetLastError());                                                                           \
  }
  if (p.few) {
    a.score = reinterpret_cast<float*>(workspace);
    a.ml = reinterpret_cast<f32x2*>(a.score + (size_t)B * cache->heads * p.rows * p.pitch);
    KSTEPS(weights_scores_kernel, dim3((unsigned)p.ranges, heads_of_all))
    hipLaunchKernelGGL(weights_sum_kernel, dim3((unsigned)((max_keys + 255) / 256), heads_of_all), dim3(256), 0, st, a);
    return (int)hipGetLastError();
  }
  a.row = reinterpret_cast<f32x2*>(workspace);
  a.ml = a.row + (size_t)T * heads;
  KSTEPS(weights_max_kernel, dim3((unsigned)(p.row_tiles * p.ranges), heads_of_all))
  if (p.ranges > 1) {
    hipLaunchKernelGGL(weights_join_kernel, dim3((unsigned)((T * heads + 255) / 256)), dim3(256), 0, st, a);
    RC_RET((int)hipGetLastError());
  }
  KSTEPS(weights_mass_kernel, dim3((unsigned)((max_keys + WEIGHT_KEYS - 1) / WEIGHT_KEYS), heads_of_all))
#undef KSTEPS
  return 0;
}
