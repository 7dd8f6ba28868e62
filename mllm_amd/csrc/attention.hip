// Attention of one token, a tree of drafted tokens or a chunk of a prompt over a paged cache, for gfx950.
//
//   o[t][h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * (q[t][h] . k_j) - m),  m = max_j,  over the keys j that token t sees:
//   the prefix of its sequence and those of the sequence's new tokens whose bit is set in its row of the tree (without a tree: itself
//   and the ones before it).
//
// The rows of one matrix product are (token, query head of the group) pairs that share a key head: with one token and four query heads a
// key head, four rows.  Everything is turned so that nothing of P leaves its lane:
//   S^T = K Q^T   v_mfma_f32_16x16x32_bf16, first operand 16 keys (a lane: 8 consecutive elements of one key), second 16 rows of Q.  Result: a
//                 lane has one row of Q (lane % 16) and four keys.  Two such products, first operand rows r = keys 8 (r / 4) + r % 4 and the same + 4,
//                 leave a lane with the eight consecutive keys 8 (lane / 16) .. + 7 of its row,
//   O^T = V^T P^T which is what the second operand of the product over 32 keys takes.  V^T comes from LDS through the transposing reads.
// A row's maximum, sum and the correction of O when the maximum grows are therefore numbers of a lane; sums over keys cross lanes twice per 32 keys
// (the maximum) and once at the end (the sum).  Scores, maxima, sums and O are fp32.
//
// Roundings: bf16 queries as they are; P to bf16 for the product with V (off by 2^-8 of each weight at most, of either sign; the sum takes P as it
// was).  fp32 queries and P enter as three bf16 parts each that add up to them (8 bits each, three products); products with fewer were off by 5e-6.
//
// A workgroup has four waves, WR along rows times 4 / WR along keys, and goes through a range of keys in tiles: 16-byte loads into registers while
// the tile before them is worked on, from there into LDS.  Rows of a tile lie there with their 16-byte pieces exclusive-ored by bits of the
// key's number, so that the 16 lanes of an operand read different banks.  Where rows and heads leave CUs idle the keys are cut into ranges,
// whose O, maximum and sum meet in the workspace; a second launch joins them.
//
// What bounds it, 32 query and 8 key heads of 128: with few rows the reading of keys and values (16 fp32 tokens over up to 8000 keys each 75 us, 341 MB: 4.5
// TB/s; a copy of 2 GB has 4.96), one token over 4097 keys (13.2 us, 16.8 MB) two launches and the loads that wait for one another in each: lengths, table, keys,
// partial results.  32 trees of 64 tokens over up to 8192 keys (256 us, 137 GFLOP, 711 MB) the matrix and the vector pipe in turns, 30 and 40 % of the
// time busy: two waves a SIMD, as 256 registers each and 64 KB of LDS a workgroup both have it; LDS is busy 30 %.  Eight trees of 29 over up to 5000 (50 us) keys and
// values at 4 TB/s and, half of the time, partial results (34 MB written and read) and starts.  A prompt of 8192 bf16 tokens 637 us, 860 TFLOP/s of what it has to compute.
#include <type_traits>

#include "item8.h"

namespace mllmhip {

typedef short at_s16x4 __attribute__((ext_vector_type(4)));
typedef short at_s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef float at_f32x4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
  const void* q;
  void* o;
  int64_t q_token, q_head, o_token, o_head;
  const uint16_t *k, *v;
  int64_t head_stride;
  uint32_t page_bytes, slot_bytes, page_end;  // page_end: bytes of a page's slots
  uint32_t step_pages, step_bytes;            // a tile's keys in whole pages and the bytes of the slots over
  uint32_t pages, page, page_mul;             // key / page = (2 key * page_mul) >> 32 >> page_shift for key < 2^31
  int page_shift;
  const int32_t* table;
  int64_t table_stride;
  int table_len;
  const int32_t *cu, *prefix;
  const uint64_t* tree;
  int64_t tree_stride;
  int words;
  int T, B, kv, group, max_tokens, row_tiles;
  int ranges, min_tiles;  // ranges that all keys are cut into (0: a sequence is never cut), tiles of a range at least
  float c;  // scale * log2 e
  float *part_o, *part_ml;  // of a sequence that is cut, [piece][its token][query head][head_dim] and [2]
  int* info;                // [B][2]: first piece and number of pieces of a sequence
};
__device__ u32x4 g_zero_row[32];  // what a page outside the cache reads as (never written)

// sequence b: its first row of q, its number of new tokens, of prefix keys and of keys
struct Seq {
  int first, n, prefix, keys;
};
__device__ __forceinline__ Seq sequence(const AttnArgs& a, int b) {
  Seq s;
  const int lo = a.cu[b], hi = min(a.cu[b + 1], a.T);
  s.first = max(lo, 0);
  s.n = max(hi - s.first, 0);
  s.prefix = max(a.prefix[b], 0);
  s.keys = (int)min((int64_t)s.prefix + s.n, (int64_t)a.table_len * a.page);
  return s;
}

// Where the keys are cut.  The tiles of all sequences, one sequence behind the other, are cut into ranges of equal length, one per workgroup (for
// every key head and tile of rows), so that workgroups have as much to do whatever the sequences' lengths are.  A range can end one sequence
// and begin another: its part of sequence b is piece range + b.  Every wave works out where its range begins, a sequence per lane.
struct Place {
  Seq s;
  int b, start, per, total;  // its number, its first tile, the tiles of a range and of all sequences
};
template <int KT>
__device__ __forceinline__ int tiles_of(const Seq& s) { return s.n > 0 ? (s.keys + KT - 1) / KT : 0; }
template <int KT>
__device__ __forceinline__ Place find_place(const AttnArgs& a, int range) {
  Place p = {{0, 0, 0, 0}, 0, 0, 0, 0};
  if (a.B == 1) {
    p.s = sequence(a, 0);
    p.total = tiles_of<KT>(p.s);
    p.per = max(a.min_tiles, (p.total + a.ranges - 1) / a.ranges);
    return p;
  }
  const int lane = threadIdx.x & 63;
  Seq mine = sequence(a, min(lane, a.B - 1));
  int total = lane < a.B ? tiles_of<KT>(mine) : 0;
  for (int b = lane + 64; b < a.B; b += 64) total += tiles_of<KT>(sequence(a, b));
#pragma unroll
  for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
  p.total = __builtin_amdgcn_readfirstlane(total);
  p.per = max(a.min_tiles, (p.total + a.ranges - 1) / a.ranges);
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    if (b0) mine = sequence(a, min(b0 + lane, a.B - 1));
    const int tiles = b0 + lane < a.B ? tiles_of<KT>(mine) : 0;
    int up = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(up, d);
      up += lane >= d ? o : 0;
    }
    const uint64_t found = __ballot(p.start + up > range * p.per);
    if (found) {
      const int at = __builtin_ctzll(found);
      p.b = b0 + at;
      p.s = Seq{__builtin_amdgcn_readlane(mine.first, at), __builtin_amdgcn_readlane(mine.n, at), __builtin_amdgcn_readlane(mine.prefix, at),
                __builtin_amdgcn_readlane(mine.keys, at)};
      p.start += __builtin_amdgcn_readlane(up - tiles, at);
      return p;
    }
    p.start += __builtin_amdgcn_readlane(up, 63);
  }
  return p;
}

__device__ __forceinline__ float larger(float x, float y) { return __builtin_elementwise_maximum(x, y); }
template <int N>  // the larger of a lane's and that of the lane N away
__device__ __forceinline__ float across(float v) {
  const u32x2 r = N == 16 ? lanes16(__float_as_uint(v)) : lanes32(__float_as_uint(v));
  return larger(__uint_as_float(r.x), __uint_as_float(r.y));
}
// 8 bf16 of a register quad as an operand
__device__ __forceinline__ at_bf16x8 frag(u32x4 v) { return __builtin_bit_cast(at_bf16x8, v); }
__device__ __forceinline__ at_f32x4 mma(at_bf16x8 x, at_bf16x8 y, at_f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, acc, 0, 0, 0); }

template <int D, int NQ, int WR, bool F32>
struct Attn {
  static constexpr int WK = 4 / WR;                      // waves along keys
  static constexpr int KT = 64;                          // keys of a tile
  static constexpr int SUB = KT / (WK * 32);             // 32-key steps of a wave per tile
  static constexpr int C = D / 8;                        // 16-byte pieces of a row
  static constexpr int NLOAD = KT / 4 / 8;               // rows of a tile that a lane loads from
  static constexpr int PARTS = F32 ? 3 : 1, PPARTS = F32 ? 3 : 1;
  static constexpr int ROWS = NQ * 16;                   // rows of a wave
  static constexpr int WAVES = D == 256 ? 1 : 2;         // per SIMD: all 512 registers for one, or 256 each
  static __device__ __forceinline__ int swz(int row) { return (C == 8) ? (row & 3) | ((row >> 3) & 1) << 2 : (row & 3) | ((row >> 3) & 3) << 2; }
};

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
// which of the keys k0 .. k0 + 7 token `token` of the sequence sees
__device__ __forceinline__ uint32_t seen_keys(const AttnArgs& a, const Seq& s, int k0, int token) {
  uint32_t see = 0;
  const int j0 = k0 - s.prefix;  // the new token that key k0 is
  if (j0 <= -8) {
    see = 0xff;
  } else if (a.tree) {  // eight bits of the token's row from bit j0 on, ones in front of bit 0
    const int lo = max(j0, 0), w = lo >> 6, in = lo & 63;
    const uint64_t* row = a.tree + (int64_t)(s.first + token) * a.tree_stride;
    uint64_t bits = w < a.words ? row[w] >> in : 0;
    if (in > 56 && w + 1 < a.words) bits |= row[w + 1] << (64 - in);
    see = (uint32_t)bits << (lo - j0) | ((1u << (lo - j0)) - 1);
  } else {
    see = (2u << min(max(token - j0, 0), 7)) - 1;  // bits 0 .. token - j0
    if (token < j0) see = 0;
  }
  const int left = s.keys - k0;
  return left >= 8 ? see & 0xff : left <= 0 ? 0 : see & ((1u << left) - 1);
}
// whether one of two bf16 is infinite or no number
__device__ __forceinline__ bool odd_pair(uint32_t v) { return ((v & 0x7f80u) == 0x7f80u) | ((v & 0x7f800000u) == 0x7f800000u); }
__device__ __forceinline__ uint32_t finite_pair(uint32_t v) {
  return ((v & 0x7f80u) == 0x7f80u ? 0u : v & 0xffffu) | ((v & 0x7f800000u) == 0x7f800000u ? 0u : v & 0xffff0000u);
}

// Infinities and NaNs among the values make that element of the rows that see them infinite or NaN, whatever the weight: it is their sum.  What the matrix products
// leave there is NaN where a weight is too small for its type (or a part of one is 0), and without them where they were taken out for rows that do not see
// them (in tiles with masks; the sum of the weights has its sign set then).  So results of either kind are looked at once more, behind everything else: a lane's elements
// d .. d + 3 of query head `head`, token `token`, where it says so in `look` (LOOK_WHOLE: among all keys, LOOK_MASKED: those of tiles with masks, the first of which has the prefix's end or the last key).  The lanes that are
// there go through the values of one result after the other together: a call of one token over 4096 keys 19 us, with a NaN among them 80 (a lane for each result: 1043).
enum { LOOK_MASKED = 1, LOOK_WHOLE = 2 };
__device__ __forceinline__ uint32_t look_at(at_f32x4 x, float sum, uint32_t sign) {
  const float most = larger(larger(fabsf(x[0]), fabsf(x[1])), larger(fabsf(x[2]), fabsf(x[3])));
  return sum != sum ? 0 : !(most < INFINITY) ? LOOK_WHOLE : sign >> 31;  // (scores that are NaN make that of the whole row)
}
template <bool F32>
__device__ __forceinline__ void put_infinities(const AttnArgs& a, const Seq& s, int b, uint32_t look, int head_, int token_, int d_) {
  const uint64_t active = __ballot(true);
  const int lanes = __popcll(active), rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(active >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)active, 0));
  const int32_t* table = a.table + b * a.table_stride;
#pragma unroll 1
  for (uint64_t left = __ballot(look); left; left &= left - 1) {
    const int who = __builtin_ctzll(left), head = __builtin_amdgcn_readlane(head_, who), token = __builtin_amdgcn_readlane(token_, who), d = __builtin_amdgcn_readlane(d_, who);
    const uint16_t* v = a.v + head / a.group * a.head_stride + d;
    const int end = a.tree ? s.keys : (int)min((int64_t)s.keys, (int64_t)s.prefix + token + 1);
    uint32_t nans = 0, above = 0, below = 0;  // which of the elements have a NaN, an infinity, one below 0
    for (int k0 = __builtin_amdgcn_readlane(look, who) == LOOK_WHOLE ? 0 : min(s.prefix, s.keys - 1) / 64 * 64; k0 < end && nans != 15; k0 += lanes) {
      const int key = min(k0 + rank, end - 1);
      const uint32_t page = __umulhi(2 * (uint32_t)key, a.page_mul) >> a.page_shift, id = (uint32_t)table[min((int)page, a.table_len - 1)];
      const uint64_t at = (uint64_t)id * a.page_bytes + (((uint32_t)key - page * a.page) * a.slot_bytes + (uint64_t)(uintptr_t)v);
      const u32x2 x = *reinterpret_cast<const __attribute__((address_space(1))) u32x2*>(id < a.pages ? at : (uint64_t)(uintptr_t)g_zero_row);
      const bool has = (odd_pair(x.x) || odd_pair(x.y)) && (seen_keys(a, s, key, token) & 1);
      if (!__ballot(has)) continue;
      const uint32_t w[4] = {x.x << 16, x.x & 0xffff0000u, x.y << 16, x.y & 0xffff0000u};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (__ballot(has && (w[e] & 0x7fffffffu) > 0x7f800000u)) nans |= 1u << e;
        if (__ballot(has && w[e] == 0x7f800000u)) above |= 1u << e;
        if (__ballot(has && w[e] == 0xff800000u)) below |= 1u << e;
      }
    }
    nans |= above & below;
    const int64_t to = (s.first + token) * a.o_token + head * a.o_head + d;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t sum = nans >> e & 1 ? 0x7fc00000u : above >> e & 1 ? 0x7f800000u : 0xff800000u;
      if ((int)(threadIdx.x & 63) == who && (nans | above | below) >> e & 1) {  // (by the lane that has stored the result)
        if (F32) reinterpret_cast<uint32_t*>(a.o)[to + e] = sum;
        else reinterpret_cast<uint16_t*>(a.o)[to + e] = (uint16_t)(sum >> 16);
      }
    }
  }
}

// The part of sequence b with keys k_begin .. k_end - 1, for key head h and row tile rt; `range` and `count` say where partial results go
template <int D, int NQ, int WR, bool F32>
__device__ __forceinline__ void attention_piece(const AttnArgs& a, const Seq& s, int b, int h, int rt, int k_begin, int k_end, int range, int count) {
  typedef Attn<D, NQ, WR, F32> P;
  constexpr int KT = P::KT, C = P::C, WK = P::WK, NLOAD = P::NLOAD, KS = D / 32, DT = D / 16;
  __shared__ __align__(16) uint16_t s_k[2 * KT * D];
  __shared__ __align__(16) uint16_t s_v[2 * KT * D];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave % WR, wk = wave / WR;
  const int col = lane & 15, g = lane >> 4;
  const int rows = s.n * a.group, row0 = rt * P::ROWS * WR;
  if (row0 >= rows) return;
  // Without a tree the tile's last token sees the most keys, and what its first one sees all of them see: keys behind the one are left out, tiles in front
  // of the other need no masks.
  int all = min(s.prefix, k_end);
  if (!a.tree) {
    int first = 0, last = s.n - 1;
    if (rows > P::ROWS * WR) {  // (a single token has no time for divisions)
      first = row0 / a.group;
      last = (min(rows, row0 + P::ROWS * WR) - 1) / a.group;
    }
    all = min(k_end - 1 - first, s.prefix) + first + 1;  // prefix + first + 1, k_end at most
    k_end = min(k_end - 1 - last, s.prefix) + last + 1;
  }
  // A lane loads 16-byte pieces p, p + 8, .. (p = lane % 8) of row lane / 8 of every eight rows.  Where a row's key is in the cache goes on from tile to
  // tile without a division: `page` numbers into the table, `in` bytes into the page.
  const int32_t* table = a.table + b * a.table_stride;
  uint32_t page[NLOAD], in[NLOAD];
  int ids[NLOAD];
  auto load_row = [&](int i) { return wave * (KT / 4) + i * 8 + lane / 8; };
#pragma unroll
  for (int i = 0; i < NLOAD; i++) {
    const uint32_t key = (uint32_t)(k_begin + load_row(i));
    page[i] = __umulhi(2 * key, a.page_mul) >> a.page_shift;
    in[i] = (key - page[i] * a.page) * a.slot_bytes;
    ids[i] = table[min((int)page[i], a.table_len - 1)];
  }
  auto next_pages = [&]() {
#pragma unroll
    for (int i = 0; i < NLOAD; i++) {
      in[i] += a.step_bytes;
      page[i] += a.step_pages;
      const bool over = in[i] >= a.page_end;
      in[i] -= over ? a.page_end : 0;
      page[i] += over;
      ids[i] = table[min((int)page[i], a.table_len - 1)];  // (behind the table: any page, never used)
    }
  };
  // Q: second operand, row `col` of every 16, elements 32 s + 8 g .. + 7
  at_bf16x8 fq[P::PARTS][NQ][KS];
  int token[NQ];
#pragma unroll
  for (int i = 0; i < NQ; i++) {
    const int r = row0 + wr * P::ROWS + i * 16 + col;
    const bool live = r < rows;
    token[i] = live ? r / a.group : 0;
    const int head = h * a.group + (live ? r - token[i] * a.group : 0);
    const int64_t at = (s.first + token[i]) * a.q_token + head * a.q_head + 8 * g;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      Item8<F32 ? MLLM_HIP_F32 : MLLM_HIP_BF16> it;
      item_load<F32 ? MLLM_HIP_F32 : MLLM_HIP_BF16>(a.q, at + 32 * ks, it);
      if (!F32) {
        fq[0][i][ks] = frag(it.r[0]);
      } else {
        float v[8];
        item_to_f32<F32 ? MLLM_HIP_F32 : MLLM_HIP_BF16>(it, v);
        uint32_t part[3][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          split2(finite(v[2 * j]), finite(v[2 * j + 1]), part[0][j], part[1][j], part[2][j]);
          // (what is no number or infinite: all in the first part)
          part[0][j] = (finite(v[2 * j]) == v[2 * j] ? part[0][j] & 0xffffu : f32_to_bf16(v[2 * j])) | (finite(v[2 * j + 1]) == v[2 * j + 1] ? part[0][j] & 0xffff0000u : (uint32_t)f32_to_bf16(v[2 * j + 1]) << 16);
        }
#pragma unroll
        for (int p = 0; p < P::PARTS; p++) fq[p][i][ks] = frag(u32x4{part[p][0], part[p][1], part[p][2], part[p][3]});
      }
    }
  }

  u32x4 rk[NLOAD][C / 8], rv[NLOAD][C / 8];
  typedef const __attribute__((address_space(1))) u32x4* global_row;  // (a select between generic pointers would be flat loads)
  const uint64_t zero = (uint64_t)(uintptr_t)g_zero_row, k_at = (uint64_t)(uintptr_t)(a.k + h * a.head_stride) + lane % 8 * 16,
                 v_less_k = (uint64_t)(uintptr_t)a.v - (uint64_t)(uintptr_t)a.k;
  auto ask_tile = [&](int k0) {
#pragma unroll
    for (int i = 0; i < NLOAD; i++) {
      const bool good = k0 + load_row(i) < k_end && (uint32_t)ids[i] < a.pages;
      const uint64_t at = (uint64_t)(uint32_t)ids[i] * a.page_bytes + (k_at + in[i]);
      const global_row kp = reinterpret_cast<global_row>(good ? at : zero), vp = reinterpret_cast<global_row>(good ? at + v_less_k : zero);
#pragma unroll
      for (int j = 0; j < C / 8; j++) {
        rk[i][j] = kp[8 * j];
        rv[i][j] = vp[8 * j];
      }
    }
    next_pages();
  };

  at_f32x4 acc[NQ][DT];
  float m[NQ], l[NQ];  // the maximum so far times c; the sum of this lane's keys
#pragma unroll
  for (int i = 0; i < NQ; i++) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; d++) acc[i][d] = at_f32x4{0.f, 0.f, 0.f, 0.f};
  }

  if (k_begin < k_end) ask_tile(k_begin);
  // Q is here from now on: a wait for it in the loops would be one for the loads of the next tile, which come behind it
#pragma unroll
  for (int p = 0; p < P::PARTS; p++)
#pragma unroll
    for (int i = 0; i < NQ; i++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++) asm volatile("" : "+v"(fq[p][i][ks]));
  bool odd = false;  // infinities or NaNs among the values of this wave's keys in tiles with masks
  // the products of a tile, which is in that half of LDS; `border`: keys that some rows do not see, or behind the last
  const bool busy = row0 + wr * P::ROWS < rows;  // (a wave without rows loads with the others and leaves its SIMD to them)
  auto work = [&](int k0, auto border_, auto half) {
    constexpr bool border = decltype(border_)::value;
#pragma unroll
    for (int u = 0; u < P::SUB; u++) {
      const int base = (u * WK + wk) * 32;  // the step's first row in the tile
      const int key0 = k0 + base;
      if (border && key0 >= k_end) break;
      at_f32x4 sa[NQ], sb[NQ];
#pragma unroll
      for (int i = 0; i < NQ; i++) sa[i] = sb[i] = at_f32x4{0.f, 0.f, 0.f, 0.f};
      const int ra = half * KT + base + 8 * (col >> 2) + (col & 3), x = P::swz(ra);
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const int at = ra * D + ((4 * ks + g) ^ x) * 8;
        const at_bf16x8 ka = frag(*reinterpret_cast<const u32x4*>(s_k + at)), kb = frag(*reinterpret_cast<const u32x4*>(s_k + at + 4 * D));
#pragma unroll
        for (int i = 0; i < NQ; i++) {
#pragma unroll
          for (int p = P::PARTS - 1; p >= 0; p--) {  // the smallest part first
            sa[i] = mma(ka, fq[p][i][ks], sa[i]);
            sb[i] = mma(kb, fq[p][i][ks], sb[i]);
          }
        }
      }
      at_bf16x8 fp[P::PPARTS][NQ];
#pragma unroll
      for (int i = 0; i < NQ; i++) {
        float y[8], top;
        auto scores = [&](const at_f32x4& a0, const at_f32x4& b0) {
#pragma unroll
          for (int j = 0; j < 4; j++) y[j] = a0[j], y[4 + j] = b0[j];
          if (border) {
            const uint32_t see = seen_keys(a, s, key0 + 8 * g, token[i]);
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = see >> j & 1 ? y[j] : -INFINITY;
          }
          // (maximum, which hands a NaN on, is one instruction for three; fmaxf quiets each of its operands first)
          top = larger(larger(larger(y[0], y[1]), larger(y[2], y[3])), larger(larger(y[4], y[5]), larger(y[6], y[7])));
          top = across<16>(top);
          top = across<32>(top) * a.c;
        };
        scores(sa[i], sb[i]);
        if (__ballot(F32 ? !(top <= m[i] + 8.f) : top > m[i] + 8.f)) {  // (weights of up to 2^8 do as well: most steps leave O alone)
          if constexpr (F32) {
            // An infinite element of a key makes a NaN with the second and third part of a query's, which may be 0: it counts with the first alone, which
            // has the sign.  Such scores, and those that are NaN anyway, are formed once more.
            if (__builtin_expect(__ballot(top != top) != 0, 0)) {
              at_f32x4 ta = {0.f, 0.f, 0.f, 0.f}, tb = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int ks = 0; ks < KS; ks++) {
                const int at = ra * D + ((4 * ks + g) ^ x) * 8;
                const u32x4 ka = *reinterpret_cast<const u32x4*>(s_k + at), kb = *reinterpret_cast<const u32x4*>(s_k + at + 4 * D);
                const at_bf16x8 fa = frag(u32x4{finite_pair(ka.x), finite_pair(ka.y), finite_pair(ka.z), finite_pair(ka.w)}),
                                fb = frag(u32x4{finite_pair(kb.x), finite_pair(kb.y), finite_pair(kb.z), finite_pair(kb.w)});
#pragma unroll
                for (int p = P::PARTS - 1; p > 0; p--) {
                  ta = mma(fa, fq[p][i][ks], ta);
                  tb = mma(fb, fq[p][i][ks], tb);
                }
                ta = mma(frag(ka), fq[0][i][ks], ta);
                tb = mma(frag(kb), fq[0][i][ks], tb);
              }
              scores(ta, tb);
            }
          }
          const float next = fmaxf(m[i], top), fix = m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[i] - next);
          m[i] = next;
          l[i] *= fix;
#pragma unroll
          for (int d = 0; d < DT; d++) acc[i][d] *= fix;
        }
        const float ref = m[i] == -INFINITY ? 0.f : m[i];  // (nothing seen yet: every p is exp2(-inf))
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = __builtin_amdgcn_exp2f(fmaf(y[j], a.c, -ref));
        l[i] += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
        if (!F32) {
          fp[0][i] = frag(u32x4{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7])});
        } else {
          uint32_t part[3][4];
#pragma unroll
          for (int j = 0; j < 4; j++) split2(y[2 * j], y[2 * j + 1], part[0][j], part[1][j], part[2][j]);
#pragma unroll
          for (int p = 0; p < P::PPARTS; p++) fp[p][i] = frag(u32x4{part[p][0], part[p][1], part[p][2], part[p][3]});
        }
      }
      // V^T: lane i of 16 asks for elements 4 (i % 4) .. + 3 of key 8 g + i / 4 and gets element i of keys 8 g .. + 3
      const int rv0 = half * KT + base + 8 * g + (col >> 2), xv = P::swz(rv0);
#pragma unroll
      for (int d = 0; d < DT; d++) {
        const int at = rv0 * D + ((2 * d + ((col & 3) >> 1)) ^ xv) * 8 + (col & 1) * 4;
        typedef __attribute__((address_space(3))) at_s16x4* lds_ptr;
        const at_s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(s_v + at));
        const at_s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(s_v + at + 4 * D));
        u32x4 vt = __builtin_bit_cast(u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        if (border) {  // a value that a row does not see must not reach it, and 0 * NaN would: such values are taken out here and come back below
          if (__ballot(odd_pair(vt.x) || odd_pair(vt.y) || odd_pair(vt.z) || odd_pair(vt.w))) {
            vt = u32x4{finite_pair(vt.x), finite_pair(vt.y), finite_pair(vt.z), finite_pair(vt.w)};
            odd = true;
          }
        }
        const at_bf16x8 fv = frag(vt);
#pragma unroll
        for (int i = 0; i < NQ; i++) {
#pragma unroll
          for (int p = P::PPARTS - 1; p >= 0; p--) acc[i][d] = mma(fv, fp[p][i], acc[i][d]);
        }
      }
    }
  };
  auto put_tile = [&](auto half) {
#pragma unroll
    for (int i = 0; i < NLOAD; i++) {
      const int row = load_row(i);
#pragma unroll
      for (int j = 0; j < C / 8; j++) {
        const int at = half * (KT * D) + row * D + ((lane % 8 + 8 * j) ^ P::swz(row)) * 8;
        *reinterpret_cast<u32x4*>(s_k + at) = rk[i][j];
        *reinterpret_cast<u32x4*>(s_v + at) = rv[i][j];
      }
    }
  };
  typedef std::integral_constant<int, 0> Lower;
  typedef std::integral_constant<int, 1> Upper;
  int k0 = k_begin;  // the tile that is worked on
  if (k_begin < k_end) {
    __syncthreads();  // what this workgroup had in LDS before has been read
    put_tile(Lower());
    if (k_begin + KT < k_end) ask_tile(k_begin + KT);
    __syncthreads();
  }
  auto turn = [&](auto border_, auto half, auto other) {
    if (busy) work(k0, border_, half);
    k0 += KT;
    if (k0 < k_end) {  // into the other half of LDS: everyone is past the tile that was there
      put_tile(other);
      if (k0 + KT < k_end) ask_tile(k0 + KT);
      __syncthreads();
    }
  };
  // Tiles of keys that every row sees, in turns whose halves of LDS are constants; then (a loop of its own: its masks would take registers from the other) the rest.
  const int plain = all - KT;  // the last tile that may begin there
  int half = 0;
  while (k0 <= plain) {
    turn(std::false_type(), Lower(), Upper());
    half = 1;
    if (k0 > plain) break;
    turn(std::false_type(), Upper(), Lower());
    half = 0;
  }
  while (k0 < k_end) {
    turn(std::true_type(), half, half ^ 1);
    half ^= 1;
  }
#pragma unroll
  for (int i = 0; i < NQ; i++) l[i] = sum32(sum16(l[i]));

  // Where a row's results go: 32-bit sizes of a row, 64-bit offsets worked out once per row.
  const int heads = a.kv * a.group;
  struct To {
    void* o;
    float* ml;
    bool part;
  };
  auto where = [&](int row) {  // of 0 .. rows - 1; o null: a token beyond the host's bound
    const int t = row / a.group, head = h * a.group + row - t * a.group;
    if (count == 1) return To{reinterpret_cast<char*>(a.o) + ((s.first + t) * a.o_token + head * a.o_head) * (F32 ? 4 : 2), nullptr, false};
    const int64_t at = ((int64_t)(range + b) * a.max_tokens + t) * heads + head;
    return To{t < a.max_tokens ? a.part_o + at * D : nullptr, a.part_ml + 2 * at, true};
  };
  // `ll`: the sum of the weights, its sign as l's.  How the result has to be looked at once more
  auto put = [&](const To& to, int d, at_f32x4 x, float mm, float ll) -> uint32_t {
    if (to.part) {
      if (!to.o) return 0;
      *reinterpret_cast<at_f32x4*>(reinterpret_cast<float*>(to.o) + d) = x;
      if (d == 0) {
        to.ml[0] = mm;
        to.ml[1] = ll;
      }
      return 0;
    }
    const float sum = fabsf(ll);
    x *= sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);  // (no key seen: zeros; a NaN stays)
    if (F32) *reinterpret_cast<at_f32x4*>(reinterpret_cast<float*>(to.o) + d) = x;
    else *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(to.o) + d) = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
    return look_at(x, sum, __float_as_uint(ll));
  };
#pragma unroll
  for (int i = 0; i < NQ; i++) l[i] = odd ? -l[i] : l[i];
  uint32_t look = 0;  // two bits for every result of a lane
  constexpr int HALF = D / 2, IT = 16 * (HALF / 4) / (WK * 64);  // (half of O at a time: four waves' rows of 256 elements would not fit)
  // The waves along keys meet in LDS, 16 rows at a time: O of a row at [row][HALF], its maximum and sum apart.
  if constexpr (WK == 1) {
#pragma unroll
    for (int i = 0; i < NQ; i++) {
      const int row = row0 + wr * P::ROWS + i * 16 + col;
      if (row >= rows) continue;
      const To to = where(row);
#pragma unroll
      for (int d = 0; d < DT; d++) look |= put(to, 16 * d + 4 * g, acc[i][d], m[i], l[i]) << 2 * (i * DT + d);
    }
  } else {
    float* so = reinterpret_cast<float*>(s_k);   // [wave][16][HALF]
    float* sm = reinterpret_cast<float*>(s_v);   // [wave][16][2]
    static_assert(4 * 16 * HALF * 4 <= KT * D * 2 && 4 * 16 * 2 * 4 <= KT * D * 2, "");
    static_assert(16 * (HALF / 4) == IT * WK * 64 && NQ * 2 * IT <= 16, "");
#pragma unroll
    for (int i = 0; i < NQ; i++) {
#pragma unroll
      for (int part = 0; part < 2; part++) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DT / 2; d++) *reinterpret_cast<at_f32x4*>(so + (wave * 16 + col) * HALF + ((4 * d + g) ^ (col & 7)) * 4) = acc[i][part * (DT / 2) + d];
        if (g == 0) {
          sm[(wave * 16 + col) * 2] = m[i];
          sm[(wave * 16 + col) * 2 + 1] = l[i];
        }
        __syncthreads();
        // the WK waves of row block w: every one of them joins a share of its 16 rows
#pragma unroll
        for (int it = 0; it < IT; it++) {
          const int e = wk * 64 + lane + it * WK * 64, r = e / (HALF / 4), p = e % (HALF / 4);
          const int row = row0 + wr * P::ROWS + i * 16 + r;
          if (row >= rows) continue;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < WK; w++) top = fmaxf(top, sm[((w * WR + wr) * 16 + r) * 2]);
          const float ref = top == -INFINITY ? 0.f : top;
          at_f32x4 x = {0.f, 0.f, 0.f, 0.f};
          float sum = 0.f;
          uint32_t sign = 0;
#pragma unroll
          for (int w = 0; w < WK; w++) {
            const int at = (w * WR + wr) * 16 + r;
            const float f = __builtin_amdgcn_exp2f(sm[at * 2] - ref);
            sum += fabsf(sm[at * 2 + 1]) * f;
            sign |= __float_as_uint(sm[at * 2 + 1]);
            x += *reinterpret_cast<const at_f32x4*>(so + at * HALF + (p ^ (r & 7)) * 4) * f;
          }
          look |= put(where(row), part * HALF + p * 4, x, top, __uint_as_float((__float_as_uint(sum) & 0x7fffffffu) | (sign & 0x80000000u))) << 2 * ((i * 2 + part) * IT + it);
        }
      }
    }
  }
  if (__builtin_expect(__ballot(look) != 0, 0)) {
#pragma unroll 1
    for (int n = 0; n < (WK == 1 ? NQ * DT : NQ * 2 * IT); n++) {
      int row, d;
      if (WK == 1) {
        row = n / DT * 16 + col;
        d = n % DT * 16 + 4 * g;
      } else {
        const int e = wk * 64 + lane + n % IT * (WK * 64);
        row = n / (2 * IT) * 16 + e / (HALF / 4);
        d = n / IT % 2 * HALF + e % (HALF / 4) * 4;
      }
      row += row0 + wr * P::ROWS;
      put_infinities<F32>(a, s, b, look >> 2 * n & 3, h * a.group + row % a.group, row / a.group, d);
    }
  }
}

template <int D, int NQ, int WR, bool F32>
__global__ __launch_bounds__(256, (Attn<D, NQ, WR, F32>::WAVES)) void attention_kernel(AttnArgs a) {
  constexpr int KT = Attn<D, NQ, WR, F32>::KT;
  // Workgroup i runs on XCD i % 8: the row tiles of a range of keys follow one another on one XCD, whose L2 they share.  The last tile comes first: without a tree it
  // has the most keys, and the shorter ones fill the end.  Prompts of 1000 (fp32), 2048, 4096 and 8192 tokens, first tile first / last tile first: 65.8 / 54.8 us,
  // 82 / 75, 231 / 187, 738 / 640; up to 1024 bf16 tokens, with a tree, and in chunks of 1024 over 8192 keys no difference.
  const int idx = blockIdx.x >> 3, rt = a.row_tiles - 1 - idx % a.row_tiles, place = (idx / a.row_tiles) * 8 + (blockIdx.x & 7);
  const int h = place % a.kv, range = place / a.kv;
  Place p = {{0, 0, 0, 0}, range, 0, 0, 0};
  int tile = 0, end;
  if (a.ranges) {
    p = find_place<KT>(a, range);
    tile = range * p.per;
    end = min(tile + p.per, p.total);
  } else {  // a sequence is a range
    if (range >= a.B) return;
    p.s = sequence(a, range);
    end = p.total = tiles_of<KT>(p.s);
  }
  while (tile < end) {
    const int tiles = tiles_of<KT>(p.s), stop = min(end, p.start + tiles);
    int count = 1;
    if (a.ranges) {
      const int first = p.start / p.per;
      count = (p.start + tiles - 1) / p.per - first + 1;
      if (h == 0 && rt == 0 && tile == p.start && threadIdx.x < 2) a.info[2 * p.b + threadIdx.x] = threadIdx.x ? count : first + p.b;
    }
    attention_piece<D, NQ, WR, F32>(a, p.s, p.b, h, rt, (tile - p.start) * KT, min((stop - p.start) * KT, p.s.keys), range, count);
    p.start += tiles;
    tile = stop;
    if (tile < end) {  // (there is a sequence with that tile)
      do p.s = sequence(a, ++p.b);
      while (tiles_of<KT>(p.s) == 0);
    }
  }
}

// Joins the pieces of a row: 16 bytes of it per lane, G groups of lanes along the pieces
template <int D, bool F32, int G>
__global__ __launch_bounds__(256) void attention_join_kernel(AttnArgs a) {
  constexpr int L = D / 4, PER = 256 / L / G;
  static_assert(PER >= 1, "");
  __shared__ at_f32x4 s_x[G > 1 ? 256 : 1];
  __shared__ float s_ml[G > 1 ? 256 / L * 2 : 1];
  const int heads = a.kv * a.group, b = blockIdx.y, tid = threadIdx.x;
  const int first = a.info[2 * b], count = a.info[2 * b + 1];
  const Seq s = sequence(a, b);
  if (s.n == 0 || count < 2) return;
  const int i = blockIdx.x * PER + tid / L % PER, group = tid / L / PER;
  const int64_t all = (int64_t)a.max_tokens * heads;
  const bool live = i < min((int64_t)s.n * heads, all);
  const int d = tid % L * 4;
  float m = -INFINITY, sum = 0.f;
  uint32_t sign = 0;  // of any piece's sum
  at_f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    const float* ml = a.part_ml + 2 * (first * all + i);
    const float* o = a.part_o + (first * all + i) * D + d;
    constexpr int U = G > 1 ? 8 : 4;  // pieces a turn; each is read where there is one (all of a turn at once: one token over 4097 keys 13.9 -> 13.0 us, eight trees of 29 over 5000, with few pieces a row, 55 -> 62)
    for (int k = group; k < count; k += U * G) {
      float mk[U], lk[U];
      at_f32x4 xk[U];
#pragma unroll
      for (int j = 0; j < U; j++) {
        const int64_t at = (int64_t)min(k + j * G, count - 1) * all;
        mk[j] = ml[2 * at];
        lk[j] = ml[2 * at + 1];
        xk[j] = *reinterpret_cast<const at_f32x4*>(o + at * D);
      }
#pragma unroll
      for (int j = 0; j < U; j++) {
        if (k + j * G >= count) break;
        const float next = fmaxf(m, mk[j]), ref = next == -INFINITY ? 0.f : next;
        const float f = __builtin_amdgcn_exp2f(m - ref), fk = __builtin_amdgcn_exp2f(mk[j] - ref);
        x = x * f + xk[j] * fk;
        sum = sum * f + fabsf(lk[j]) * fk;
        sign |= __float_as_uint(lk[j]);
        m = next;
      }
    }
  }
  if constexpr (G > 1) {
    s_x[tid] = x;
    if (d == 0) {
      s_ml[tid / L * 2] = m;
      s_ml[tid / L * 2 + 1] = __uint_as_float((__float_as_uint(sum) & 0x7fffffffu) | (sign & 0x80000000u));
    }
    __syncthreads();
    if (group) return;
    const int row = tid / L;
    float top = -INFINITY;
    for (int k = 0; k < G; k++) top = fmaxf(top, s_ml[(k * PER + row) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
    x = at_f32x4{0.f, 0.f, 0.f, 0.f};
    sum = 0.f;
    for (int k = 0; k < G; k++) {
      const float f = __builtin_amdgcn_exp2f(s_ml[(k * PER + row) * 2] - ref), part = s_ml[(k * PER + row) * 2 + 1];
      x += s_x[tid + k * PER * L] * f;
      sum += fabsf(part) * f;
      sign |= __float_as_uint(part);
    }
  }
  if (!live) return;
  x *= sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
  const int64_t token = i / heads, to = (s.first + token) * a.o_token + (i - token * heads) * a.o_head + d;
  if (F32) *reinterpret_cast<at_f32x4*>(reinterpret_cast<float*>(a.o) + to) = x;
  else *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(a.o) + to) = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
  const uint32_t look = look_at(x, sum, sign);
  if (__builtin_expect(__ballot(look) != 0, 0)) put_infinities<F32>(a, s, b, look, (int)(i - token * heads), (int)token, d);
}

// ---- host side ------------------------------------------------------------------------------------------------------------
struct AttnPlan {
  int nq, wr, row_tiles, ranges, min_tiles;
};
// Rows of a workgroup by the rows there are (tokens times query heads of a key head): 32 rows a wave (16 with fp32 queries, whose parts, and with heads of 256,
// whose O takes the registers), waves along rows before waves along keys.  Keys are cut while there are under 1024 workgroups without that and more keys
// than four tiles and than two ranges have, into ranges that give every CU two workgroups, of twice as many keys as rows at least: what a range hands over
// is rows, what it reads keys.  One token of 32 heads, uncut / cut, us: 128 keys 7.8 / 10.1, 256 9.4 / 10.5, 320 10.4 / 11.1, 500 13.2 / 10.4, 768 16.8 / 10.5:
// the second launch, which joins the ranges, is what cutting costs (4 of them).  Prompts with no more keys than two ranges: four of 300 tokens 21.5 / 38,
// eight chunks of 30 over 500 keys 24.8 / 30.0, one of 128 over 500 24.7 / 22.4; up to four ranges: one of 128 over 1000 39 / 25.
// From 1024 workgroups on, cutting evens out unequal lengths.  Single tokens over up to n keys, a quarter of it at least: 128 of them, n 8000, 524 / 464, 6144 406 / 361,
// 4097 274 / 253, 2000 136 / 132, 1000 74 / 77; 64 trees of 64, n 8192, 582 / 535, 4097 308 / 295, 2000 170 / 176.  Of equal lengths it costs 1 to 2 %: 128 tokens over 4097 keys
// 379 / 382, 64 trees 388 / 397, and its workspace (64 trees: 102 MB).  So it is done from 6144 keys on, where it gains 8 to 12 %, up to two row tiles (a prompt's ranges
// are not alike) and 4096 workgroups, from where it gains as little as it may cost: 512 single tokens over up to 8000 keys 1870 / 1820, 4097 967 / 950, 4097 each 1445 / 1489.
static AttnPlan attention_plan(bool f32, int64_t B, int heads, int kv, int64_t max_tokens, int64_t max_keys, int D) {
  AttnPlan p;
  const int64_t rows = max_tokens * (heads / kv);
  p.nq = rows <= 32 || f32 || D == 256 ? 1 : 2;
  p.wr = rows <= 32 || (rows <= 64 && p.nq == 2) ? 2 : 4;
  const int64_t per = (int64_t)p.nq * 16 * p.wr;
  const int64_t row_tiles = (rows + per - 1) / per;
  p.row_tiles = (int)row_tiles;
  const int kt = 64;
  p.min_tiles = (int)((2 * (rows < per ? rows : per) + kt - 1) / kt);
  const int64_t most = B * ((max_keys + p.min_tiles * kt - 1) / (p.min_tiles * kt)), wanted = (512 + kv * row_tiles - 1) / (kv * row_tiles);
  const int64_t uncut = B * kv * row_tiles;
  const bool full = uncut >= 1024 && (row_tiles > 2 || max_keys < 6144 || uncut >= 4096);
  p.ranges = full || max_keys <= (p.min_tiles > 2 ? 2 * p.min_tiles : 4) * kt ? 0 : (int)(wanted < most ? wanted : most);
  if (p.ranges <= 1 && B == 1) p.ranges = 0;
  if (row_tiles > 2 && p.ranges <= B) p.ranges = 0;  // (no more workgroups than without: 16 prompts of 600 tokens of two key heads of 64 24 us, cut 43)
  return p;
}
// partial results of every piece, and of every sequence where its pieces are
static size_t attention_room(const AttnPlan& p, int64_t B, int heads, int64_t max_tokens, int D) {
  return p.ranges ? ((size_t)(p.ranges + B) * max_tokens * heads * (D + 2) + 2 * B) * sizeof(float) : 0;
}
static bool attention_sizes(int dtype, int64_t T, int64_t B, int heads, int kv, int head_dim, int64_t max_tokens, int64_t max_keys) {
  return (dtype == MLLM_HIP_F32 || dtype == MLLM_HIP_BF16) && T >= 0 && B >= 0 && heads >= 1 && kv >= 1 && max_tokens >= 0 && max_keys >= 0;
}
static bool attention_shape(int64_t T, int64_t B, int heads, int kv, int head_dim, int64_t max_tokens, int64_t max_keys) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) && heads % kv == 0 && heads <= 65536 && T <= 0x7fffffff / heads && B <= 0x7fffffff / heads &&
         max_tokens <= 0x7fffffff / heads && max_keys <= 0x7fff0000;
}

}  // namespace mllmhip

using namespace mllmhip;

MLLM_API size_t mllm_hip_attention_paged_workspace_bytes(int dtype, int64_t T, int64_t B, int heads, int kv_heads, int head_dim, int64_t max_tokens,
                                                         int64_t max_keys) {
  if (!attention_sizes(dtype, T, B, heads, kv_heads, head_dim, max_tokens, max_keys) || !attention_shape(T, B, heads, kv_heads, head_dim, max_tokens, max_keys)) return 0;
  if (T == 0 || B == 0 || max_tokens == 0) return 0;
  if (max_tokens > T) max_tokens = T;
  const AttnPlan p = attention_plan(dtype == MLLM_HIP_F32, B, heads, kv_heads, max_tokens, max_keys, head_dim);
  return attention_room(p, B, heads, max_tokens, head_dim);
}

MLLM_API int mllm_hip_attention_paged(const mllm_hip_heads* q, int dtype, int64_t T, const mllm_hip_kv_cache* cache, const int32_t* block_table,
                                      int64_t table_stride, int64_t table_len, const int32_t* cu_tokens, const int32_t* prefix, int64_t B,
                                      int64_t max_tokens, int64_t max_keys, const uint64_t* tree, int64_t tree_stride, int64_t tree_words, float scale,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !cache || table_len < 0 || tree_words < 0 || !(scale > 0.f) || scale > 2e38f || cache->pages < 1 || cache->page_size < 1) return MLLM_HIP_E_BADARG;
  if (!attention_sizes(dtype, T, B, q->heads, cache->heads, cache->head_dim, max_tokens, max_keys)) return MLLM_HIP_E_BADARG;
  if (!attention_shape(T, B, q->heads, cache->heads, cache->head_dim, max_tokens, max_keys) || cache->pages > 0x7fffffff / cache->page_size ||
      table_len > 0x7fff0000 / cache->page_size || tree_words > 0x1ffffff || cache->page_stride < 0 || cache->slot_stride < 0 || cache->page_stride > 0x7fffffff ||
      cache->slot_stride > 0x3fffffff / cache->page_size ||
      (cache->slot_stride == 0 && cache->page_size > 1))
    return MLLM_HIP_E_SHAPE;
  if (T == 0 || B == 0 || max_tokens == 0) return 0;
  if (max_tokens > T) max_tokens = T;
  if (!q->x || !q->y || !cache->k || !cache->v || !block_table || !cu_tokens || !prefix || table_len < 1) return MLLM_HIP_E_BADARG;
  const int wide = dtype == MLLM_HIP_F32 ? 4 : 2;
  auto al = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  auto whole = [&](int64_t stride) { return stride * wide % 16 == 0; };
  if (!al(q->x, 16) || !al(q->y, 16) || !al(cache->k, 16) || !al(cache->v, 16) || !whole(q->x_token_stride) || !whole(q->x_head_stride) || !whole(q->y_token_stride) ||
      !whole(q->y_head_stride) || cache->page_stride % 8 || cache->slot_stride % 8 || cache->head_stride % 8 || !al(block_table, 4) || !al(cu_tokens, 4) || !al(prefix, 4) ||
      !al(tree, 8) || !al(workspace, 16))
    return MLLM_HIP_E_ALIGN;
  if (q->x == q->y || !own_places(*q, T)) return MLLM_HIP_E_BADARG;
  const bool f32 = dtype == MLLM_HIP_F32;
  const int heads = q->heads, D = cache->head_dim;
  AttnPlan p = attention_plan(f32, B, heads, cache->heads, max_tokens, max_keys, D);
  if (B * (table_len * cache->page_size / 64 + 1) > 0x1fffffff) p.ranges = 0;  // (tiles are counted in 32 bits)
  const size_t need = attention_room(p, B, heads, max_tokens, D);
  if (need && (!workspace || workspace_bytes < need)) return MLLM_HIP_E_BADARG;
  const int64_t pieces = p.ranges + B, groups = ((p.ranges ? p.ranges : B) * cache->heads + 7) / 8 * 8;
  if (groups > 0xffffff / p.row_tiles) return MLLM_HIP_E_SHAPE;
  AttnArgs a = {};
  a.q = q->x;
  a.o = q->y;
  a.q_token = q->x_token_stride;
  a.q_head = q->x_head_stride;
  a.o_token = q->y_token_stride;
  a.o_head = q->y_head_stride;
  a.k = reinterpret_cast<const uint16_t*>(cache->k);
  a.v = reinterpret_cast<const uint16_t*>(cache->v);
  a.page_bytes = (uint32_t)(cache->page_stride * 2);
  a.slot_bytes = (uint32_t)(cache->slot_stride * 2);
  a.page_end = cache->page_size == 1 ? 1 : (uint32_t)(cache->page_size * cache->slot_stride * 2);  // (a page of one slot: `in` stays 0)
  const int kt = 64;
  a.step_pages = (uint32_t)(kt / cache->page_size);
  a.step_bytes = (uint32_t)(kt % cache->page_size * cache->slot_stride * 2);
  a.head_stride = cache->head_stride;
  a.pages = (uint32_t)cache->pages;
  a.page = (uint32_t)cache->page_size;
  // key / page for key < 2^31: with 2^s >= page the multiplier ceil(2^(31 + s) / page) is off by less than 2^s / 2^31 of a key
  int s = 0;
  while ((1ll << s) < cache->page_size) s++;
  a.page_mul = (uint32_t)(((1ull << (31 + s)) + cache->page_size - 1) / cache->page_size);
  a.page_shift = s;
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_len = (int)table_len;
  a.cu = cu_tokens;
  a.prefix = prefix;
  a.tree = tree;
  a.tree_stride = tree_stride;
  a.words = (int)tree_words;
  a.T = (int)T;
  a.B = (int)B;
  a.kv = cache->heads;
  a.group = heads / cache->heads;
  a.max_tokens = (int)max_tokens;
  a.row_tiles = p.row_tiles;
  a.ranges = p.ranges;
  a.min_tiles = p.min_tiles;
  a.c = scale * 1.44269504088896341f;
  a.part_o = reinterpret_cast<float*>(workspace);
  if (p.ranges) {
    a.part_ml = a.part_o + (size_t)pieces * max_tokens * heads * D;
    a.info = reinterpret_cast<int*>(a.part_ml + (size_t)pieces * max_tokens * heads * 2);
  }
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(groups * p.row_tiles));
  const int form = p.nq * 10 + p.wr;
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, a); };
#define ATTN(D_, NQ_, WR_, F_) \
  case NQ_ * 10 + WR_: go(attention_kernel<D_, NQ_, WR_, F_>); break;
#define ATTN_D(D_)                                                                            \
  if (f32) switch (form) { ATTN(D_, 1, 2, true) ATTN(D_, 1, 4, true) }                        \
  else switch (form) { ATTN(D_, 1, 2, false) ATTN(D_, 2, 2, false) ATTN(D_, 2, 4, false) }
  if (D == 64) {
    ATTN_D(64)
  } else if (D == 128) {
    ATTN_D(128)
  } else if (f32) {
    switch (form) { ATTN(256, 1, 2, true) ATTN(256, 1, 4, true) }
  } else {
    switch (form) { ATTN(256, 1, 2, false) ATTN(256, 1, 4, false) }
  }
#undef ATTN_D
#undef ATTN
  RC_RET((int)hipGetLastError());
  if (p.ranges) {
    // lanes along the ranges where a sequence has many of them: one row of 17 ranges by lanes that take them in turn was 11 us of dependent loads
    const bool many = p.ranges >= 8 * B;
    const int per = many ? 1 : 256 / (D / 4);
    const dim3 jgrid((unsigned)((max_tokens * heads + per - 1) / per), (unsigned)B);
    auto join = [&](auto kern) { hipLaunchKernelGGL(kern, jgrid, dim3(256), 0, st, a); };
#define JOIN(D_, F_)                                               \
  if (many) join(attention_join_kernel<D_, F_, 1024 / D_>);        \
  else join(attention_join_kernel<D_, F_, 1>)
    if (D == 64) {
      if (f32) { JOIN(64, true); } else { JOIN(64, false); }
    } else if (D == 128) {
      if (f32) { JOIN(128, true); } else { JOIN(128, false); }
    } else {
      if (f32) { JOIN(256, true); } else { JOIN(256, false); }
    }
#undef JOIN
  }
  return (int)hipGetLastError();
}
