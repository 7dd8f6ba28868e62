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
//   Up to 16 rows whose scores fit into 64 KB, of few keys or many sequences: the two in one launch, a workgroup a key head, scores in LDS.
// No atomics: what a key gets is summed by one wave in one order.
//
// What bounds it.  Tokens: memory (a token of 16 sequences over up to 8000 keys, 32 query and 8 key heads of 128, 57 us: scores 47, of which keys arrive at 3.7 TB/s (a load of a wave is 64 bytes of each of 16 keys; attention over an encoder's states, whose loads are whole rows, has 4.1 to 4.4), sums 9.5; neither more ranges, nor ranges of equal
// length over all sequences, nor heads of a range on one XCD changed that; 64 sequences over up to 3800 keys 88, 3.7 TB/s too, whether 64 or 128 KB a CU are on their way).  More rows: matrix instructions, three parts of fp32 queries in both passes (32 tokens of six sequences over up to 7000 keys 76 to 81 us:
// parts 5.6, maxima 35, join 4.7, weights 40; the bytes alone would take 12, the products at a library's rate 25; bf16 queries 54 where the products take 11, 500 of them over 4000 keys 68 to 70 where they take 27).  Storing the scores of many rows instead of forming them twice would write and read more bytes than that.
#include <type_traits>

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
  f32x2* row;    // [T][heads]: maximum (times c) and 1 / sum of all keys; null where what needs them joins the ranges'
  float* part;   // [split][B][kv][pitch]: what keys get of a part of the rows
  int splits;
  uint16_t* parts;  // fp32 queries as three bf16 parts, [3][T][heads][D]
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

__device__ __forceinline__ uint32_t page_of(const WeightArgs& a, int key) { return __umulhi(2 * (uint32_t)key, a.page_mul) >> a.page_shift; }
// elements 32 ks + 8 g .. + 7 of key `key`, which is in page `id`
template <int KS>
__device__ __forceinline__ void load_key_of(const WeightArgs& a, uint64_t k_at, int id, int key, int g, u32x4 (&r)[KS]) {
  const bool good = (uint32_t)id < a.pages;
  const uint64_t at = good ? k_at + (uint64_t)(uint32_t)id * a.page_bytes + ((uint32_t)key - page_of(a, key) * a.page) * a.slot_bytes : (uint64_t)(uintptr_t)g_no_key;
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    const int e = 32 * ks + 8 * g;
    r[ks] = *reinterpret_cast<const __attribute__((address_space(1))) u32x4*>(e < a.D ? at + e * 2 : (uint64_t)(uintptr_t)g_no_key);
  }
}
template <int KS>
__device__ __forceinline__ void load_key(const WeightArgs& a, const int32_t* table, uint64_t k_at, int key, bool there, int g, u32x4 (&r)[KS]) {
  load_key_of<KS>(a, k_at, there ? table[page_of(a, key)] : -1, key, g, r);
}

// Rows of C 16-byte pieces lie in LDS with their pieces exclusive-ored by bits of the row's number, so that 16 rows' pieces of one number are in different banks.
template <int C>
__device__ __forceinline__ int swizzle(int row) {
  return C == 8 ? (row >> 1) & 7 : C == 12 ? (row >> 2) & 3 : row & 15;
}
// what a key gets
__device__ __forceinline__ void put_mass(const WeightArgs& a, const WeightSeq& s, int b, int h, int key, float v) {
  if (key >= a.mass_len) return;
  float* mass = a.mass + b * a.mass_seq + h * a.mass_head + key;
  *mass = key < s.prefix && a.decay != 0.f ? a.decay * *mass + v : v;
}

// Scores (times 1) of 16 keys and 16 rows
template <int KS, bool F32>
__device__ __forceinline__ at_f32x4 raw_scores(const u32x4 (&k)[KS], const at_bf16x8 (&q)[KS][F32 ? 3 : 1]) {
  at_f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < KS; ks++)
#pragma unroll
    for (int p = (F32 ? 3 : 1) - 1; p >= 0; p--) s = mma(frag(k[ks]), q[ks][p], s);  // the smallest part first
  return s;
}
// With fp32 queries an infinite element of a key makes a NaN with the second and third part of a query's, which may be 0: it counts with the first alone, which has the sign.  Scores that
// are NaN are formed once more like this.  (The keys go through an asm: what follows from them would else be worked out in front of the branch that leads here, and be most of the instructions.)
template <int KS>
__device__ __forceinline__ at_f32x4 scores_again(const u32x4 (&k)[KS], const at_bf16x8 (&q)[KS][3]) {
  at_f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    u32x4 x = k[ks];
    asm volatile("" : "+v"(x));
    const at_bf16x8 f = frag(u32x4{finite_pair(x.x), finite_pair(x.y), finite_pair(x.z), finite_pair(x.w)});
    s = mma(f, q[ks][2], s);
    s = mma(f, q[ks][1], s);
    s = mma(frag(x), q[ks][0], s);
  }
  return s;
}
template <int KS, bool F32>
__device__ __forceinline__ at_f32x4 key_scores(const u32x4 (&k)[KS], const at_bf16x8 (&q)[KS][F32 ? 3 : 1]) {
  at_f32x4 s = raw_scores<KS, F32>(k, q);
  if constexpr (F32) {
    const float all = (s[0] + s[1]) + (s[2] + s[3]);
    if (__builtin_expect(__ballot(all != all) != 0, 0)) s = scores_again<KS>(k, q);
  }
  return s;
}
// Rows r0 .. r0 + 15 of a sequence as an operand: row `col` of lane col.  MADE: the parts of fp32 queries are in the workspace.
template <int KS, bool F32, bool MADE = false>
__device__ __forceinline__ void load_rows(const WeightArgs& a, const WeightSeq& s, int h, int r, int rows, int g, at_bf16x8 (&q)[KS][F32 ? 3 : 1]) {
  const bool live = r < rows;
  const int token = live ? r / a.group : 0, head = h * a.group + (live ? r - token * a.group : 0);
  if constexpr (MADE) {
    const int64_t heads = a.kv * a.group, at = ((s.first + token) * heads + head) * a.D + 8 * g;
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int p = 0; p < 3; p++)
        q[ks][p] = frag(live && 32 * ks + 8 * g < a.D ? *reinterpret_cast<const u32x4*>(a.parts + p * a.T * heads * a.D + at + 32 * ks) : u32x4{0, 0, 0, 0});
    return;
  }
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
// a lane's scores of 16 keys from k0 on, -inf where its row does not see them
template <int KS, bool F32>
__device__ __forceinline__ at_f32x4 seen_scores(const u32x4 (&k)[KS], const at_bf16x8 (&q)[KS][F32 ? 3 : 1], int seen) {
  at_f32x4 y = key_scores<KS, F32>(k, q);
#pragma unroll
  for (int j = 0; j < 4; j++) y[j] = j < seen ? y[j] : -INFINITY;
  return y;
}

template <int KS, bool F32>
__global__ __launch_bounds__(256) void weights_scores_kernel(WeightArgs a) {
  __shared__ f32x2 s_ml[4][16];
  constexpr int U = KS == 8 ? 1 : 2, STEP = 64 * U;  // sixteens of keys of a wave at a time; keys of a workgroup
  const int h = blockIdx.y % a.kv, b = blockIdx.y / a.kv, range = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const WeightSeq s = weight_sequence(a, b);
  const int rows = min(s.n * a.group, a.rows);
  if (rows == 0) return;
  const int per = ((s.keys + a.ranges - 1) / a.ranges + 63) / 64 * 64, begin = range * per, end = min(begin + per, s.keys);
  const int32_t* table = a.table + b * a.table_stride;
  const uint64_t k_at = (uint64_t)(uintptr_t)(a.k + h * a.head_stride);
  // Keys are on their way while the ones before them are worked on, and the pages of those behind.
  int ids[U];
  u32x4 next[U][KS];
  const int first = begin + wave * 16 * U + col;
  auto ask_ids = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; u++) ids[u] = k0 + 16 * u < end ? table[page_of(a, k0 + 16 * u)] : -1;
  };
  auto ask = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; u++) load_key_of<KS>(a, k_at, ids[u], k0 + 16 * u, g, next[u]);
    ask_ids(k0 + STEP);
  };
  ask_ids(first);
  ask(first);
  at_bf16x8 q[KS][F32 ? 3 : 1];
  load_rows<KS, F32>(a, s, h, col, rows, g, q);
  const int token = col < rows ? col / a.group : -1, sees = token < 0 ? 0 : min(s.prefix + token + 1, end);
  float m = -INFINITY, l = 0.f;
  float* score = a.score + ((int64_t)blockIdx.y * a.rows + col) * a.pitch;
  for (int k0 = begin + wave * 16 * U; k0 < end; k0 += STEP) {
    u32x4 k[U][KS];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++) k[u][ks] = next[u][ks];
    if (k0 + STEP < end) ask(k0 + STEP + col);
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (k0 + 16 * u >= end) break;
      const at_f32x4 y = seen_scores<KS, F32>(k[u], q, sees - (k0 + 16 * u + 4 * g));
      if (col < a.rows) *reinterpret_cast<at_f32x4*>(score + k0 + 16 * u + 4 * g) = y;
      take(m, l, y, a.c);
    }
  }
  join_lanes(m, l);
  if (g == 0) s_ml[wave][col] = f32x2{m, l};
  __syncthreads();
  if (threadIdx.x < a.rows) {
    for (int w = 1; w < 4; w++) join(m, l, s_ml[w][col].x, s_ml[w][col].y);
    a.ml[((int64_t)range * gridDim.y + blockIdx.y) * a.rows + col] = f32x2{m, l};
  }
}

// R: at least the rows.  What a key reads is asked for in front of the joining of the ranges' maxima and sums.
template <int R>
__global__ __launch_bounds__(256) void weights_sum_kernel(WeightArgs a) {
  __shared__ f32x2 s_part[256 / R][R];
  __shared__ f32x2 s_row[R];
  const int h = blockIdx.y % a.kv, b = blockIdx.y / a.kv, tid = threadIdx.x, key = blockIdx.x * 256 + tid;
  const float* score = a.score + (int64_t)blockIdx.y * a.rows * a.pitch + min(key, a.pitch - 1);
  float y[R];
#pragma unroll
  for (int r = 0; r < R; r++) y[r] = score[(int64_t)min(r, a.rows - 1) * a.pitch];  // (of keys that are not there: any numbers, never used)
  const int r = tid % R, group = tid / R;
  float m = -INFINITY, l = 0.f;
  if (r < a.rows) {
    constexpr int U = 4;
    for (int i = group; i < a.ranges; i += U * (256 / R)) {
      f32x2 x[U];
#pragma unroll
      for (int u = 0; u < U; u++) x[u] = a.ml[((int64_t)min(i + u * (256 / R), a.ranges - 1) * gridDim.y + blockIdx.y) * a.rows + r];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (i + u * (256 / R) < a.ranges) join(m, l, x[u].x, x[u].y);
    }
  }
  const WeightSeq s = weight_sequence(a, b);
  if (s.n == 0 || blockIdx.x * 256 >= s.keys) return;
  s_part[group][r] = f32x2{m, l};
  __syncthreads();
  if (tid < R) {
    for (int i = 1; i < 256 / R && i < a.ranges; i++) join(m, l, s_part[i][tid].x, s_part[i][tid].y);
    s_row[tid] = final_row(m, l);
  }
  __syncthreads();
  if (key >= s.keys) return;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < R; i++) {
    const float p = __builtin_amdgcn_exp2f(fmaf(y[i], a.c, -s_row[i].x)) * s_row[i].y;
    sum += i < a.rows && key <= s.prefix + i / a.group ? p : 0.f;  // (a row without a number has none for keys that it sees)
  }
  put_mass(a, s, b, h, key, sum);
}

// The whole of it in one launch: a workgroup has a key head of a sequence, scores stay in LDS.
enum { WEIGHT_LDS = 16 * 964 };  // floats: with what else there is less than 64 KB
template <int KS, bool F32>
__global__ __launch_bounds__(512) void weights_one_kernel(WeightArgs a) {
  extern __shared__ __align__(16) float s_score[];  // [rows][pitch]
  __shared__ f32x2 s_ml[8][16];
  __shared__ f32x2 s_row[16];
  const int h = blockIdx.x % a.kv, b = blockIdx.x / a.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const WeightSeq s = weight_sequence(a, b);
  const int rows = min(s.n * a.group, a.rows);
  if (rows == 0) return;
  const int32_t* table = a.table + b * a.table_stride;
  const uint64_t k_at = (uint64_t)(uintptr_t)(a.k + h * a.head_stride);
  // Keys are on their way while the ones before them are worked on, and the page of those behind.
  auto page_at = [&](int key) { return key < s.keys ? table[page_of(a, key)] : -1; };
  const int first = wave * 16 + col;
  int id = page_at(first);
  u32x4 next[KS];
  load_key_of<KS>(a, k_at, id, first, g, next);
  id = page_at(first + 128);
  at_bf16x8 q[KS][F32 ? 3 : 1];
  load_rows<KS, F32>(a, s, h, col, rows, g, q);
  const int token = col < rows ? col / a.group : -1, sees = token < 0 ? 0 : min(s.prefix + token + 1, s.keys);
  float m = -INFINITY, l = 0.f;
  for (int k0 = wave * 16; k0 < s.keys; k0 += 128) {
    u32x4 k[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) k[ks] = next[ks];
    if (k0 + 128 < s.keys) {
      load_key_of<KS>(a, k_at, id, k0 + 128 + col, g, next);
      id = page_at(k0 + 256 + col);
    }
    const at_f32x4 y = seen_scores<KS, F32>(k, q, sees - (k0 + 4 * g));
    if (col < rows) *reinterpret_cast<at_f32x4*>(s_score + col * a.pitch + k0 + 4 * g) = y;
    take(m, l, y, a.c);
  }
  join_lanes(m, l);
  if (g == 0) s_ml[wave][col] = f32x2{m, l};
  __syncthreads();
  if (threadIdx.x < 16) {
    for (int w = 1; w < 8; w++) join(m, l, s_ml[w][col].x, s_ml[w][col].y);
    s_row[col] = final_row(m, l);
  }
  __syncthreads();
  for (int key = threadIdx.x; key < s.keys; key += 512) {
    float sum = 0.f;
    for (int r = 0; r < rows; r++) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s_score[r * a.pitch + key], a.c, -s_row[r].x)) * s_row[r].y;
      sum += key <= s.prefix + r / a.group ? p : 0.f;
    }
    put_mass(a, s, b, h, key, sum);
  }
}

// ---- more rows ------------------------------------------------------------------------------------------------------------
// fp32 queries as three bf16 parts, once for all that read them
__global__ __launch_bounds__(256) void weights_parts_kernel(WeightArgs a) {
  const int pieces = a.D / 8, heads = a.kv * a.group;
  const int64_t all = (int64_t)a.T * heads * pieces, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  const int64_t row = i / pieces, token = row / heads;
  at_bf16x8 part[3];
  query_parts<true>(a.q, token * a.q_token + (row - token * heads) * a.q_head + (i - row * pieces) * 8, true, part);
#pragma unroll
  for (int p = 0; p < 3; p++) *reinterpret_cast<at_bf16x8*>(a.parts + (p * all + i) * 8) = part[p];
}

// Maxima and sums: four waves, WR along rows times 4 / WR along keys, 64 keys in LDS at a time, the next ones on their way.
enum { WEIGHT_TILE = 64 };
// rows of a wave, in sixteens (fp32 queries of 256 elements take 96 registers for sixteen)
static constexpr int weight_nq(int ks, bool f32) { return ks == 8 && f32 ? 1 : 2; }

template <int KS, int WR, bool F32>
__global__ __launch_bounds__(256, 2) void weights_max_kernel(WeightArgs a) {
  constexpr int NQ = weight_nq(KS, F32), DP = KS * 32, C = DP / 8, KT = WEIGHT_TILE, NLOAD = KT * C / 256, WK = 4 / WR, NB = KT / 16 / WK, PARTS = F32 ? 3 : 1;
  __shared__ __align__(16) uint16_t s_k[2 * KT * DP];
  __shared__ f32x2 s_ml[4][NQ * 16];
  // Workgroup i runs on XCD i % 8: the row tiles of a range of keys follow one another on one XCD, whose L2 they share.
  const int idx = blockIdx.x >> 3, rt = idx % a.row_tiles, place = (idx / a.row_tiles) * 8 + (blockIdx.x & 7);
  const int h = place % a.kv, range = place / a.kv % a.ranges, b = place / a.kv / a.ranges;
  if (b >= a.B) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave % WR, wk = wave / WR, col = lane & 15, g = lane >> 4;
  const WeightSeq s = weight_sequence(a, b);
  const int rows = s.n * a.group, row0 = rt * (WR * NQ * 16);
  if (row0 >= rows) return;
  const int first = row0 / a.group, last = (min(rows, row0 + WR * NQ * 16) - 1) / a.group;
  const int per = ((s.keys + a.ranges - 1) / a.ranges + KT - 1) / KT * KT, begin = range * per;
  const int end = min(min(begin + per, s.keys), s.prefix + last + 1);  // (keys behind the last token are seen by none of these rows)
  const int plain = min(end, s.prefix + first + 1) - KT;               // the last tile that may begin there and needs no masks
  const int32_t* table = a.table + b * a.table_stride;
  const int real = a.D / 8;
  int row_of[NLOAD], to[NLOAD], ids[NLOAD];
  bool has[NLOAD];
  const uint64_t k_at = (uint64_t)(uintptr_t)(a.k + h * a.head_stride);
#pragma unroll
  for (int i = 0; i < NLOAD; i++) {
    const int e = i * 256 + tid, r = e / C, p = e % C;
    row_of[i] = r;
    has[i] = p < real;
    to[i] = r * DP + (p ^ swizzle<C>(r)) * 8;
    if (!has[i]) *reinterpret_cast<u32x4*>(s_k + to[i]) = *reinterpret_cast<u32x4*>(s_k + KT * DP + to[i]) = u32x4{0, 0, 0, 0};
  }
  auto ask_ids = [&](int k0) {
#pragma unroll
    for (int i = 0; i < NLOAD; i++) {
      const int key = k0 + row_of[i];
      ids[i] = key < end && has[i] ? table[page_of(a, key)] : -1;
    }
  };
  u32x4 rk[NLOAD];
  auto ask_tile = [&](int k0) {
#pragma unroll
    for (int i = 0; i < NLOAD; i++) {
      const uint32_t key = (uint32_t)(k0 + row_of[i]), id = (uint32_t)ids[i];
      const uint64_t at = k_at + (uint64_t)id * a.page_bytes + ((key - page_of(a, (int)key) * a.page) * a.slot_bytes + (i * 256 + tid) % C * 16);
      rk[i] = *reinterpret_cast<const __attribute__((address_space(1))) u32x4*>(id < a.pages ? at : (uint64_t)(uintptr_t)g_no_key);
    }
    ask_ids(k0 + KT);
  };
  auto put_tile = [&](int half) {
#pragma unroll
    for (int i = 0; i < NLOAD; i++)
      if (has[i]) *reinterpret_cast<u32x4*>(s_k + half * (KT * DP) + to[i]) = rk[i];
  };
  at_bf16x8 q[NQ][KS][PARTS];
  int token[NQ];
  float m[NQ], l[NQ];
  if (begin < end) {
    ask_ids(begin);
    ask_tile(begin);
  }
#pragma unroll
  for (int i = 0; i < NQ; i++) {
    const int r = row0 + (wr * NQ + i) * 16 + col;
    load_rows<KS, F32, F32>(a, s, h, r, rows, g, q[i]);
    token[i] = r < rows ? r / a.group : -1;
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  const bool busy = row0 + wr * NQ * 16 < rows;
  auto work = [&](int k0, auto border_, int half) {
    constexpr bool border = decltype(border_)::value;
    at_f32x4 y[NB][NQ];
    auto load = [&](int u, u32x4 (&k)[KS]) {
      const int row = half * KT + (u * WK + wk) * 16 + col, x = swizzle<C>(row);
#pragma unroll
      for (int ks = 0; ks < KS; ks++) k[ks] = *reinterpret_cast<const u32x4*>(s_k + row * DP + ((4 * ks + g) ^ x) * 8);
    };
    auto mask = [&](int u, int i) {
      if (!border) return;
      const int seen = token[i] < 0 ? 0 : min(s.prefix + token[i] + 1, end) - (k0 + (u * WK + wk) * 16 + 4 * g);
#pragma unroll
      for (int j = 0; j < 4; j++) y[u][i][j] = j < seen ? y[u][i][j] : -INFINITY;
    };
    auto highest = [&](int i) {
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < NB; u++) top = larger(larger(y[u][i][0], y[u][i][1]), larger(larger(y[u][i][2], y[u][i][3]), top));
      return top;
    };
#pragma unroll
    for (int u = 0; u < NB; u++) {
      u32x4 k[KS];
      load(u, k);
#pragma unroll
      for (int i = 0; i < NQ; i++) {
        y[u][i] = raw_scores<KS, F32>(k, q[i]);
        mask(u, i);
      }
    }
#pragma unroll
    for (int i = 0; i < NQ; i++) {
      float top = highest(i);  // (a NaN is handed on)
      if constexpr (F32) {
        if (__builtin_expect(__ballot(top != top) != 0, 0)) {
#pragma unroll
          for (int u = 0; u < NB; u++) {
            u32x4 k[KS];
            load(u, k);
            y[u][i] = scores_again<KS>(k, q[i]);
            mask(u, i);
          }
          top = highest(i);
        }
      }
      const float next = larger(m[i], top * a.c), ref = next == -INFINITY ? 0.f : next;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < NB; u++)
#pragma unroll
        for (int j = 0; j < 4; j++) sum += __builtin_amdgcn_exp2f(fmaf(y[u][i][j], a.c, -ref));
      l[i] = fmaf(l[i], __builtin_amdgcn_exp2f(m[i] - ref), sum);
      m[i] = next;
    }
  };
  if (begin < end) {
    put_tile(0);
    if (begin + KT < end) ask_tile(begin + KT);
    __syncthreads();
  }
  int half = 0;
  for (int k0 = begin; k0 < end; k0 += KT, half ^= 1) {
    if (busy) {
      if (k0 <= plain) work(k0, std::false_type(), half);
      else work(k0, std::true_type(), half);
    }
    if (k0 + KT < end) {
      put_tile(half ^ 1);
      if (k0 + 2 * KT < end) ask_tile(k0 + 2 * KT);
      __syncthreads();
    }
  }
  const int heads = a.kv * a.group;
#pragma unroll
  for (int i = 0; i < NQ; i++) join_lanes(m[i], l[i]);
  if constexpr (WK > 1) {  // the waves along keys
#pragma unroll
    for (int i = 0; i < NQ; i++)
      if (g == 0) s_ml[wave][i * 16 + col] = f32x2{m[i], l[i]};
    __syncthreads();
    if (wk) return;
#pragma unroll
    for (int i = 0; i < NQ; i++)
#pragma unroll
      for (int w = 1; w < WK; w++) join(m[i], l[i], s_ml[w * WR + wr][i * 16 + col].x, s_ml[w * WR + wr][i * 16 + col].y);
  }
#pragma unroll
  for (int i = 0; i < NQ; i++) {
    if (g || token[i] < 0) continue;
    const int64_t at = (int64_t)(s.first + token[i]) * heads + h * a.group + (row0 + (wr * NQ + i) * 16 + col - token[i] * a.group);
    if (a.ranges == 1) a.row[at] = final_row(m[i], l[i]);
    else a.ml[(int64_t)range * a.T * heads + at] = f32x2{m[i], l[i]};
  }
}

__global__ __launch_bounds__(256) void weights_join_kernel(WeightArgs a) {
  const int64_t all = (int64_t)a.T * a.kv * a.group, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  float m = -INFINITY, l = 0.f;
  constexpr int U = 8;
  for (int r = 0; r < a.ranges; r += U) {  // (rows of no sequence: any numbers, never used)
    f32x2 x[U];
#pragma unroll
    for (int u = 0; u < U; u++) x[u] = a.ml[min(r + u, a.ranges - 1) * all + i];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (r + u < a.ranges) join(m, l, x[u].x, x[u].y);
  }
  a.row[i] = final_row(m, l);
}

// The weights: a wave has NK * 16 keys in registers, rows go by in LDS, 32 at a time (16 of 256 elements), the next ones on their way.  Where keys leave CUs idle rows are cut into
// `splits`, whose sums a last launch adds.
// FEW: 64 keys a workgroup where those of the other form leave CUs idle and rows are too few to be split (one sequence of 16 tokens over 1000 keys, groups of four: 21.4 -> 17.8 us, four of 30 fp32 tokens over 800
// 38 -> 33, but 500 tokens over 4000 75 -> 91).  It joins the maxima and sums of up to eight ranges of keys itself (16 over 1000 16.1 -> 14.1; the registers that takes would cost the other form a wave: 6 x 32 fp32
// tokens over up to 7000 83 -> 89).
enum { WEIGHT_JOIN = 8 };
template <int KS, bool F32, bool FEW>
struct Mass {
  static constexpr int MOST = KS < 8 ? 4 : F32 ? 1 : 2, NK = FEW ? 1 : MOST, RT = KS == 8 ? 16 : 32, KEYS = 4 * NK * 16;
};
template <int KS, bool F32, bool FEW>
__global__ __launch_bounds__(256, 2) void weights_mass_kernel(WeightArgs a) {
  typedef Mass<KS, F32, FEW> P;
  constexpr int NK = P::NK, RT = P::RT, DP = KS * 32, C = DP / 8, PARTS = F32 ? 3 : 1, NL = (RT * C + 255) / 256;
  __shared__ __align__(16) uint16_t s_q[2][PARTS][RT * DP];
  __shared__ f32x2 s_row[2][RT];
  const int h = blockIdx.y % a.kv, b = blockIdx.y / a.kv, split = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, g = lane >> 4;
  const WeightSeq s = weight_sequence(a, b);
  const int rows = s.n * a.group, kg = blockIdx.x * P::KEYS, k0 = kg + wave * NK * 16;
  if (rows == 0 || kg >= s.keys) return;
  const int per = ((rows + a.splits - 1) / a.splits + RT - 1) / RT * RT, begin = max(split * per, max(kg - s.prefix, 0) * a.group / RT * RT), end = min(split * per + per, rows);
  // Sixteens of rows from row `plain` on, plain_rows of them, need no masks: each sees all of the wave's keys, and all sixteen are there.  (One that is not would add what its zeros make of an infinite
  // element of a key, which is no number.)
  const int plain = max(k0 + NK * 16 - 1 - s.prefix, 0) * a.group;
  const uint32_t plain_rows = max(end - 15 - plain, 0);
  const int heads = a.kv * a.group;
  // rows r0 .. r0 + RT - 1 on their way, 8 elements a piece
  u32x4 it[NL][PARTS];
  f32x2 factor[FEW ? WEIGHT_JOIN : 1];
  auto ask_rows = [&](int r0) {
#pragma unroll
    for (int i = 0; i < NL; i++) {
      const int e = i * 256 + tid, r = r0 + e / C, p = e % C;
      const bool there = e < RT * C && r < end && p * 8 < a.D;
      const int token = there ? r / a.group : 0, head = h * a.group + (there ? r - token * a.group : 0);
#pragma unroll
      for (int j = 0; j < PARTS; j++) {
        it[i][j] = u32x4{0, 0, 0, 0};
        if (!there) continue;
        if (F32) it[i][j] = *reinterpret_cast<const u32x4*>(a.parts + (((int64_t)j * a.T + s.first + token) * heads + head) * a.D + p * 8);
        else it[i][j] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(a.q) + (s.first + token) * a.q_token + head * a.q_head + p * 8);
      }
    }
    if (tid < RT) {
      const int r = r0 + tid, token = r / a.group;
      const int64_t at = (int64_t)(s.first + token) * heads + h * a.group + (r - token * a.group);
      factor[0] = r < end ? (!FEW || a.row ? a.row[at] : a.ml[at]) : f32x2{0.f, 0.f};
      if (FEW && !a.row) {
#pragma unroll
        for (int i = 1; i < (FEW ? WEIGHT_JOIN : 1); i++) factor[i] = r < end && i < a.ranges ? a.ml[(int64_t)i * a.T * heads + at] : f32x2{-INFINITY, 0.f};
      }
    }
  };
  auto put_rows = [&](int half) {
#pragma unroll
    for (int i = 0; i < NL; i++) {
      const int e = i * 256 + tid, r = e / C, p = e % C;
      if (RT * C % 256 && e >= RT * C) break;
#pragma unroll
      for (int j = 0; j < PARTS; j++) *reinterpret_cast<u32x4*>(&s_q[half][j][r * DP + (p ^ swizzle<C>(r)) * 8]) = it[i][j];
    }
    if (tid < RT) {
      if (FEW && !a.row) {
        float m = factor[0].x, l = factor[0].y;
#pragma unroll
        for (int i = 1; i < (FEW ? WEIGHT_JOIN : 1); i++) join(m, l, factor[i].x, factor[i].y);
        factor[0] = final_row(m, l);
      }
      s_row[half][tid] = factor[0];
    }
  };
  if (begin < end) ask_rows(begin);
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
  if (begin < end) put_rows(0);
  if (begin + RT < end) ask_rows(begin + RT);
  __syncthreads();
  int half = 0;
  for (int r0 = begin; r0 < end; r0 += RT, half ^= 1) {
#pragma unroll 1
    for (int rb = 0; rb < RT / 16; rb++) {
      const int r = r0 + rb * 16;
      if (r >= end) break;
      at_f32x4 y[NK];
#pragma unroll
      for (int i = 0; i < NK; i++) y[i] = at_f32x4{0.f, 0.f, 0.f, 0.f};
      const int x = swizzle<C>(rb * 16 + col);
      auto query = [&](int ks, int p) { return *reinterpret_cast<const at_bf16x8*>(&s_q[half][p][(rb * 16 + col) * DP + ((4 * ks + g) ^ x) * 8]); };
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
#pragma unroll
        for (int p = PARTS - 1; p >= 0; p--) {  // the smallest part first
          const at_bf16x8 q = query(ks, p);
#pragma unroll
          for (int i = 0; i < NK; i++) y[i] = mma(frag(k[i][ks]), q, y[i]);
        }
      }
      if constexpr (F32) {  // (as in scores_again)
        float all = 0.f;
#pragma unroll
        for (int i = 0; i < NK; i++) all += (y[i][0] + y[i][1]) + (y[i][2] + y[i][3]);
        if (__builtin_expect(__ballot(all != all) != 0, 0)) {  // (infinities of both signs make one too: formed once more to no harm)
#pragma unroll
          for (int i = 0; i < NK; i++) {
            y[i] = at_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
              u32x4 f4 = k[i][ks];
              asm volatile("" : "+v"(f4));
              const at_bf16x8 f = frag(u32x4{finite_pair(f4.x), finite_pair(f4.y), finite_pair(f4.z), finite_pair(f4.w)});
              y[i] = mma(f, query(ks, 2), y[i]);
              y[i] = mma(f, query(ks, 1), y[i]);
              y[i] = mma(frag(f4), query(ks, 0), y[i]);
            }
          }
        }
      }
      const f32x2 row = s_row[half][rb * 16 + col];
      if ((uint32_t)(r - plain) < plain_rows) {
#pragma unroll
        for (int i = 0; i < NK; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) sum[i][j] = fmaf(__builtin_amdgcn_exp2f(fmaf(y[i][j], a.c, -row.x)), row.y, sum[i][j]);
      } else {
        const int token = r + col < end ? (r + col) / a.group : -1;
#pragma unroll
        for (int i = 0; i < NK; i++) {
          const int seen = token < 0 ? 0 : s.prefix + token + 1 - (k0 + i * 16 + 4 * g);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float p = __builtin_amdgcn_exp2f(fmaf(y[i][j], a.c, -row.x)) * row.y;
            sum[i][j] += j < seen ? p : 0.f;  // (a row without a number has none for keys that it sees)
          }
        }
      }
    }
    if (r0 + RT < end) {
      put_rows(half ^ 1);
      if (r0 + 2 * RT < end) ask_rows(r0 + 2 * RT);
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < NK; i++) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float v = group_sum<16>(sum[i][j]);
      const int key = k0 + i * 16 + 4 * g + j;
      if (col != j || key >= s.keys) continue;
      if (a.splits > 1) a.part[((int64_t)split * gridDim.y + blockIdx.y) * a.pitch + key] = v;
      else put_mass(a, s, b, h, key, v);
    }
  }
}

__global__ __launch_bounds__(256) void weights_add_kernel(WeightArgs a) {
  const int h = blockIdx.y % a.kv, b = blockIdx.y / a.kv, key = blockIdx.x * 256 + threadIdx.x;
  const WeightSeq s = weight_sequence(a, b);
  if (s.n == 0 || key >= s.keys) return;
  float sum = 0.f;
  for (int i = 0; i < a.splits; i++) sum += a.part[((int64_t)i * gridDim.y + blockIdx.y) * a.pitch + key];
  put_mass(a, s, b, h, key, sum);
}

// ---- host side ------------------------------------------------------------------------------------------------------------
struct WeightPlan {
  bool few, one, few_keys;
  int rows, pitch, ranges, row_tiles, wr, splits, keys;
};
// Up to 16 rows (an operand's): 16 sequences of four tokens with groups of four over 4000 keys 35 us, as more rows 56.
// One launch of those, a workgroup a key head, where scores fit and either keys are few or every CU has a head.  One token, groups of four, one launch / two: one sequence over 200 keys 5.9 / 8.8 us, eight over 600 9.3 / 9.5, over 960
// 11.8 / 11.5; 32 over 1200 15.8 / 19.8, over 3800 45 / 50; 64 over 3800 89 / 103; but 24 over 3800 38.9 / 36.2, 16 over 3800 35.5 / 25.5.
// Ranges of keys of two launches: workgroups for 1024 of tokens, 512 of more rows (16 x 1 over up to 8000 keys with 512 / 1024 / 2048 58.6 / 56.7 / 54.8, a sequence of 4 over 4000 12.9 / 13.5 / 12.6; 6 x 32 fp32
// over up to 7000 with 256 / 512 / 1024 91 / 83 / 87, 2 x 100 over 3000 66 / 59 / 67), of 256 keys or, of more rows and 257 to 1024 keys, 128 (16 over 1000 17.8 -> 15.5, 2 x 60 over 500 23.1 -> 21.5, but 8 x 8 over 700
// 17.5 -> 17.8, and over 8000 29.7 -> 33).  Where keys alone give fewer than 512 workgroups rows are split as well: 500 tokens over 4000 keys 73 us, unsplit 116.
static WeightPlan weight_plan(bool f32, int64_t B, int heads, int kv, int D, int64_t max_tokens, int64_t max_keys) {
  WeightPlan p = {};
  const int64_t rows = max_tokens * (heads / kv);
  p.few = rows <= 16;
  p.rows = p.few ? (int)rows : 0;
  p.pitch = (int)((max_keys + 63) / 64 * 64);
  p.one = p.few && (p.pitch + 4) * rows <= WEIGHT_LDS && (max_keys <= 960 || B * kv >= 256);
  if (p.one) p.pitch += 4;  // (rows begin in banks of their own)
  const int64_t wave = weight_nq(D > 128 ? 8 : 4, f32) * 16;
  p.wr = rows <= wave ? 1 : rows <= 2 * wave ? 2 : 4;
  p.row_tiles = p.few ? 1 : (int)((rows + p.wr * wave - 1) / (p.wr * wave));
  const int64_t uncut = B * kv * p.row_tiles, least = p.few || max_keys <= 256 || max_keys > 1024 ? 256 : 128, most = (max_keys + least - 1) / least, wanted = p.few ? (1023 + uncut) / uncut : (511 + uncut) / uncut;
  p.ranges = (int)(uncut >= 1024 || most < 2 ? 1 : wanted < most ? wanted : most);
  const int most_keys = D <= 128 ? Mass<4, false, false>::KEYS : f32 ? Mass<8, true, false>::KEYS : Mass<8, false, false>::KEYS, few_keys = Mass<4, false, true>::KEYS;
  p.few_keys = !p.few && most_keys > few_keys && B * kv * ((max_keys + most_keys - 1) / most_keys) < 256 && rows <= 256;
  p.keys = p.few_keys ? few_keys : most_keys;
  const int64_t groups = B * kv * ((max_keys + p.keys - 1) / p.keys), parts = (rows + 127) / 128, split = (511 + groups) / groups;
  p.splits = (int)(p.few || groups >= 512 || parts < 2 ? 1 : split < parts ? split : parts);
  return p;
}
static size_t weight_room(const WeightPlan& p, bool f32, int64_t T, int64_t B, int heads, int kv, int D) {
  if (p.one) return 0;
  if (p.few) return ((size_t)B * kv * p.rows * p.pitch + (size_t)p.ranges * B * kv * p.rows * 2) * sizeof(float);
  return ((size_t)(p.ranges > 1 ? p.ranges + 1 : 1) * T * heads * 2 + (p.splits > 1 ? (size_t)p.splits * B * kv * p.pitch : 0)) * sizeof(float) + (f32 ? (size_t)T * heads * D * 6 : 0) + 16;
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
  return weight_room(weight_plan(dtype == MLLM_HIP_F32, B, heads, kv_heads, head_dim, max_tokens, max_keys), dtype == MLLM_HIP_F32, T, B, heads, kv_heads, head_dim);
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
  const WeightPlan p = weight_plan(f32, B, heads, cache->heads, D, max_tokens, max_keys);
  const size_t need = weight_room(p, f32, T, B, heads, cache->heads, D);
  if (need && (!workspace || workspace_bytes < need)) return MLLM_HIP_E_BADARG;
  const int64_t groups = (B * cache->heads * p.ranges + 7) / 8 * 8;
  if (groups > 0xffffff / p.row_tiles) return MLLM_HIP_E_SHAPE;
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
#define KSTEPS(GRID_, ...)                                                              \
  {                                                                                     \
    auto go = [&](auto ks, auto f) {                                                    \
      constexpr int KS = decltype(ks)::value;                                           \
      constexpr bool F32 = decltype(f)::value;                                          \
      hipLaunchKernelGGL((__VA_ARGS__), GRID_, dim3(256), 0, st, a);                    \
    };                                                                                  \
    auto by_type = [&](auto ks) { if (f32) go(ks, std::true_type()); else go(ks, std::false_type()); }; \
    if (D <= 64) by_type(std::integral_constant<int, 2>());                             \
    else if (D <= 96) by_type(std::integral_constant<int, 3>());                        \
    else if (D <= 128) by_type(std::integral_constant<int, 4>());                       \
    else by_type(std::integral_constant<int, 8>());                                     \
    RC_RET((int)hipGetLastError());                                                     \
  }
  if (p.one) {
    // (blocks of 512 threads: the launches below have 256)
    const size_t lds = (size_t)p.rows * p.pitch * sizeof(float);
    auto one = [&](auto ks) {
      constexpr int KS = decltype(ks)::value;
      if (f32) hipLaunchKernelGGL((weights_one_kernel<KS, true>), dim3(heads_of_all), dim3(512), lds, st, a);
      else hipLaunchKernelGGL((weights_one_kernel<KS, false>), dim3(heads_of_all), dim3(512), lds, st, a);
    };
    if (D <= 64) one(std::integral_constant<int, 2>());
    else if (D <= 96) one(std::integral_constant<int, 3>());
    else if (D <= 128) one(std::integral_constant<int, 4>());
    else one(std::integral_constant<int, 8>());
    return (int)hipGetLastError();
  }
  if (p.few) {
    a.score = reinterpret_cast<float*>(workspace);
    a.ml = reinterpret_cast<f32x2*>(a.score + (size_t)B * cache->heads * p.rows * p.pitch);
    KSTEPS(dim3((unsigned)p.ranges, heads_of_all), weights_scores_kernel<KS, F32>)
    const dim3 sums((unsigned)((max_keys + 255) / 256), heads_of_all);
    if (p.rows <= 2) hipLaunchKernelGGL(weights_sum_kernel<2>, sums, dim3(256), 0, st, a);
    else if (p.rows <= 4) hipLaunchKernelGGL(weights_sum_kernel<4>, sums, dim3(256), 0, st, a);
    else if (p.rows <= 8) hipLaunchKernelGGL(weights_sum_kernel<8>, sums, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(weights_sum_kernel<16>, sums, dim3(256), 0, st, a);
    return (int)hipGetLastError();
  }
  const bool joined = p.few_keys && p.ranges > 1 && p.ranges <= WEIGHT_JOIN;
  f32x2* const room = reinterpret_cast<f32x2*>(workspace);
  a.row = joined ? nullptr : room;
  a.ml = room + (size_t)T * heads;
  a.part = reinterpret_cast<float*>(room + (size_t)(p.ranges > 1 ? p.ranges + 1 : 1) * T * heads);
  a.splits = p.splits;
  if (f32) {
    const uintptr_t behind = reinterpret_cast<uintptr_t>(a.part) + (p.splits > 1 ? (size_t)p.splits * B * cache->heads * p.pitch * sizeof(float) : 0);
    a.parts = reinterpret_cast<uint16_t*>((behind + 15) / 16 * 16);
    hipLaunchKernelGGL(weights_parts_kernel, dim3((unsigned)((T * heads * (D / 8) + 255) / 256)), dim3(256), 0, st, a);
    RC_RET((int)hipGetLastError());
  }
  const dim3 grid((unsigned)(groups * p.row_tiles));
  if (p.wr == 1) KSTEPS(grid, weights_max_kernel<KS, 1, F32>)
  else if (p.wr == 2) KSTEPS(grid, weights_max_kernel<KS, 2, F32>)
  else KSTEPS(grid, weights_max_kernel<KS, 4, F32>)
  if (p.ranges > 1 && !joined) {
    hipLaunchKernelGGL(weights_join_kernel, dim3((unsigned)((T * heads + 255) / 256)), dim3(256), 0, st, a);
    RC_RET((int)hipGetLastError());
  }
  const dim3 mass_grid((unsigned)((max_keys + p.keys - 1) / p.keys), heads_of_all, (unsigned)p.splits);
  if (p.few_keys) KSTEPS(mass_grid, weights_mass_kernel<KS, F32, KS < 8 || !F32>)
  else KSTEPS(mass_grid, weights_mass_kernel<KS, F32, false>)
#undef KSTEPS
  if (p.splits > 1) {
    hipLaunchKernelGGL(weights_add_kernel, dim3((unsigned)((max_keys + 255) / 256), heads_of_all), dim3(256), 0, st, a);
    RC_RET((int)hipGetLastError());
  }
  return 0;
}
