// Attention over an encoder's states, which have another length than the queries and no order among them, for gfx950.
//
//   o[t][h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * (q[t][h] . k_j) - m),  m = max_j,  over all keys j of the sequence that token t is of.
//
// The products are turned as over the paged cache: S^T = K Q^T leaves a lane with one row of Q (a pair of a token and a query head of the group that shares a
// key head) and eight consecutive keys, which is what the second operand of O^T = V^T P^T takes.  Scores, maxima, sums and O are fp32; P is rounded to bf16 for
// the product with V (off by 2^-8 of each weight at most, of either sign), fp32 queries and their P enter as three bf16 parts each.
//
// Two forms.  Up to 64 rows of a sequence and key head or keys of a sequence, fp32 queries and heads of more than 128 elements: cross_kernel, on products of 16 x 16 x 32.  A workgroup has four waves, WR along rows times
// 4 / WR along keys, and goes through the keys in tiles of 64: 16-byte loads into registers while the tile before them is worked on, from there into LDS.  Heads of 72 or 80 elements take three
// steps of 32 in the first product (zeros behind them) and five tiles of 16 in the second.  More bf16 rows: cross_wide_kernel, on products of 32 x 32 x 16, keys and values from memory to LDS directly.
// Where rows, heads and sequences leave CUs idle the keys are cut into pieces, whose O, maximum and sum meet in the workspace; a second launch joins them.
//
// What bounds it.  Few rows: memory, behind the chain of two launches (64 sequences of one token over 1601 keys, 32 query and 8 key heads of 128, 74 to 79 us: 4.1 to 4.4 TB/s where a copy of 2 GB has 5.18; four
// fp32 tokens over 1601 keys 15.4, of which the join takes 3.9).  64 x 64 windows of 160 images, 16 heads of 80: 20 us, 3.9 TB/s.  Many rows: matrix and vector instructions, which share a SIMD's issue and overlap only
// in part, at the clock that both leave (1.8 GHz): 4900 tokens over 4900 keys, 16 heads of 80, 157 us (780 TFLOP/s; a product of 8192^3 has 1229), 3 x 700 tokens over up to 6404 keys, 32 heads of 128, 155 to 180
// (730 to 850), 10 000 over 10 000, four query heads a key head, 550 (930).  The wide form's matrix pipes are busy 43 to 48 % of the time, and none of its LDS reads meets a taken bank.
// Next tile's scores between this one's exponents (a third more registers) and four waves a SIMD (spills) were no faster; equal shares of the keys of all tiles per CU, whose parts are joined, cost 24 us to join.
#include <type_traits>

#include "attention_common.h"

namespace mllmhip {

struct CrossArgs {
  const void* q;
  void* o;
  int64_t q_token, q_head, o_token, o_head;
  const uint16_t *k, *v;
  int64_t k_head, v_head;
  uint32_t k_bytes, v_bytes;  // from a key to the next
  const int32_t *cu, *first, *count;
  int64_t keys;  // rows of k and v
  int T, B, kv, group, D, max_tokens, row_tiles, rows_of_tile, pieces, min_tiles;
  int whole, tiles;         // row tiles whose keys are not cut, and all of them
  float c;                  // scale * log2 e
  float *part_o, *part_ml;  // of the tiles that are cut, [piece][tile][row][D], [2]
};
__device__ u32x4 g_no_state[32];  // what keys behind the last read as (never written)

struct CrossSeq {
  int first, n;  // rows of q
  int64_t key;   // its first key
  int keys;
};
__device__ __forceinline__ CrossSeq cross_sequence(const CrossArgs& a, int b) {
  CrossSeq s;
  const int lo = max(a.cu[b], 0), hi = min(a.cu[b + 1], a.T);
  s.first = lo;
  s.n = min(max(hi - lo, 0), a.max_tokens);
  s.key = min((int64_t)max(a.first[b], 0), a.keys);
  s.keys = (int)min((int64_t)max(a.count[b], 0), a.keys - s.key);
  return s;
}
// What a workgroup has: row tile `tile` of all (those of a sequence's key head one behind the other), and of its keys piece `piece`
struct CrossPlace {
  CrossSeq s;
  int b, h, tile, piece, pieces, row0, rows, k_begin, k_end;
};
// of a tile that is cut: tiles of 64 keys in a piece, and pieces
__device__ __forceinline__ void cut(const CrossArgs& a, int keys, int& per, int& pieces) {
  const int tiles = (keys + 63) / 64;
  per = max(a.min_tiles, (tiles + a.pieces - 1) / a.pieces);
  pieces = max(1, (tiles + per - 1) / per);
}
// Row tile `tile` in the order of workgroups.  Of several row tiles a head, key heads, which have equal work, go round the XCDs (workgroup i runs on XCD i % 8), the row tiles of one, which share its keys, stay on theirs;
// of one each, neighbouring heads, whose states share cache lines, are on one.
__device__ __forceinline__ void cross_tile(const CrossArgs& a, int tile, int& place, int& rt) {
  if (a.whole == 0 || a.row_tiles == 1) {
    const int j = a.whole ? xcd_run(tile, a.tiles) : tile;
    rt = j % a.row_tiles;
    place = j / a.row_tiles;
    return;
  }
  const int heads = a.B * a.kv, round = heads / 8 * 8 * a.row_tiles;
  if (tile < round) {
    const int q = tile >> 3;
    rt = q % a.row_tiles;
    place = q / a.row_tiles * 8 + (tile & 7);
  } else {
    const int j = round + xcd_run(tile - round, heads * a.row_tiles - round);
    rt = j % a.row_tiles;
    place = j / a.row_tiles;
  }
}
__device__ __forceinline__ bool cross_place(const CrossArgs& a, CrossPlace& p) {
  const int i = blockIdx.x;
  p.piece = 0;
  p.tile = i;
  if (i >= a.whole) {  // (a multiple of 8, or all)
    const int j = xcd_run(i - a.whole, (a.tiles - a.whole) * a.pieces);
    p.tile = a.whole + j / a.pieces;
    p.piece = j % a.pieces;
  }
  int place, rt;
  cross_tile(a, p.tile, place, rt);
  p.h = place % a.kv;
  p.b = place / a.kv;
  p.s = cross_sequence(a, p.b);
  p.rows = p.s.n * a.group;
  p.row0 = rt * a.rows_of_tile;
  p.pieces = 1;
  p.k_begin = 0;
  p.k_end = p.s.keys;
  if (i >= a.whole && a.pieces > 1) {
    int per;
    cut(a, p.s.keys, per, p.pieces);
    p.k_begin = p.piece * per * 64;
    p.k_end = min(p.k_begin + per * 64, p.s.keys);
  }
  return p.row0 < p.rows && p.piece < p.pieces;
}

// Elements d .. d + 3 of a row's result: O, its maximum and sum go to the workspace where keys are cut
template <bool F32>
__device__ __forceinline__ void cross_put(const CrossArgs& a, const CrossPlace& p, int row, int token, int head, int d, at_f32x4 x, float m, float sum) {
  if (d >= a.D) return;
  if (p.pieces > 1) {
    const int64_t at = ((int64_t)p.piece * (a.tiles - a.whole) + (p.tile - a.whole)) * a.rows_of_tile + (row - p.row0);
    *reinterpret_cast<at_f32x4*>(a.part_o + at * a.D + d) = x;
    if (d == 0) {
      a.part_ml[2 * at] = m;
      a.part_ml[2 * at + 1] = sum;
    }
    return;
  }
  x *= sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);  // (no key: zeros; a NaN stays)
  const int64_t at = (p.s.first + token) * a.o_token + head * a.o_head + d;
  if (F32) *reinterpret_cast<at_f32x4*>(reinterpret_cast<float*>(a.o) + at) = x;
  else *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(a.o) + at) = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
}

// ONE: sequences of one tile of keys, as the host says.  Half the LDS and registers for no second tile leave room for more workgroups a CU (heads of 80: five of bf16, four of fp32; two to three of the other form), whose loads and stores overlap:
// 160 windows of 64, 16 heads of 80, 23.8 -> 20.8 us, 300 of 49 and 72 33.6 -> 25.6, 100 fp32 ones of 80 30.2 -> 22.9.  More rows than 64 as well, which the other form has by 128: 4000 tokens over 64 keys, heads of 128,
// 14.6 -> 13.5, 20 x 300 19.1 -> 17.4 (4 x 400 over 40 8.3 both).
template <int DP, int DT, int WR, bool F32, bool ONE>
struct Cross {
  static constexpr int WK = 4 / WR;          // waves along keys
  static constexpr int KT = 64;              // keys of a tile
  static constexpr int SUB = KT / (WK * 32); // 32-key steps of a wave per tile
  static constexpr int C = DP / 8;           // 16-byte pieces of a row
  static constexpr int NLOAD = KT * C / 256; // pieces of a tile that a lane loads, of keys and of values
  static constexpr int PARTS = F32 ? 3 : 1;
  static constexpr int WAVES = DP == 256 ? 1 : ONE ? 3 : 2;
  // Rows of 8 and of 16 or 32 pieces begin in the same banks every second or every row; rows of 12 every fourth.
  static __device__ __forceinline__ int swz(int row) {
    return C == 12 ? (row >> 3) & 3 : C == 8 ? (row & 3) | ((row >> 3) & 1) << 2 : (row & 3) | ((row >> 3) & 3) << 2;
  }
};

template <int DP, int DT, int WR, bool F32, bool ONE>
__global__ __launch_bounds__(256, (Cross<DP, DT, WR, F32, ONE>::WAVES)) void cross_kernel(CrossArgs a) {
  typedef Cross<DP, DT, WR, F32, ONE> P;
  constexpr int KT = P::KT, C = P::C, WK = P::WK, NLOAD = P::NLOAD, KS = DP / 32, PARTS = P::PARTS;
  constexpr int HALVES = ONE ? 1 : 2;  // of LDS: tiles in turn
  __shared__ __align__(16) uint16_t s_k[HALVES * KT * DP];
  __shared__ __align__(16) uint16_t s_v[HALVES * KT * DP];
  CrossPlace place;
  if (!cross_place(a, place)) return;
  const CrossSeq& s = place.s;
  const int h = place.h, rows = place.rows, row0 = place.row0, k_begin = place.k_begin, k_end = place.k_end;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave % WR, wk = wave / WR;
  const int col = lane & 15, g = lane >> 4;

  // Piece i of a lane's: piece at[i] % C of row at[i] / C of a tile.  Pieces behind a head's end are zeros in LDS from the beginning.
  const int real = a.D / 8;
  int row_of[NLOAD], to[NLOAD];
  uint32_t koff[NLOAD], voff[NLOAD];
  bool has[NLOAD];
#pragma unroll
  for (int i = 0; i < NLOAD; i++) {
    const int e = i * 256 + tid, r = e / C, p = e % C;
    row_of[i] = r;
    has[i] = p < real;
    to[i] = r * DP + (p ^ P::swz(r)) * 8;
    koff[i] = r * a.k_bytes + p * 16;
    voff[i] = r * a.v_bytes + p * 16;
    if (!has[i]) {
#pragma unroll
      for (int half = 0; half < HALVES; half++) {
        *reinterpret_cast<u32x4*>(s_k + half * KT * DP + to[i]) = u32x4{0, 0, 0, 0};
        *reinterpret_cast<u32x4*>(s_v + half * KT * DP + to[i]) = u32x4{0, 0, 0, 0};
      }
    }
  }
  typedef const __attribute__((address_space(1))) u32x4* global_row;
  const uint64_t zero = (uint64_t)(uintptr_t)g_no_state;
  const uint64_t k_at = (uint64_t)(uintptr_t)(a.k + h * a.k_head) + s.key * a.k_bytes, v_at = (uint64_t)(uintptr_t)(a.v + h * a.v_head) + s.key * a.v_bytes;
  u32x4 rk[NLOAD], rv[NLOAD];
  auto ask_tile = [&](int k0) {
#pragma unroll
    for (int i = 0; i < NLOAD; i++) {
      const bool good = k0 + row_of[i] < k_end && has[i];
      rk[i] = *reinterpret_cast<global_row>(good ? k_at + (uint64_t)k0 * a.k_bytes + koff[i] : zero);
      rv[i] = *reinterpret_cast<global_row>(good ? v_at + (uint64_t)k0 * a.v_bytes + voff[i] : zero);
    }
  };
  auto put_tile = [&](auto half) {
#pragma unroll
    for (int i = 0; i < NLOAD; i++) {
      if (!has[i]) continue;
      *reinterpret_cast<u32x4*>(s_k + half * (KT * DP) + to[i]) = rk[i];
      *reinterpret_cast<u32x4*>(s_v + half * (KT * DP) + to[i]) = rv[i];
    }
  };
  if (k_begin < k_end) ask_tile(k_begin);

  // Q: second operand, row `col`, elements 32 s + 8 g .. + 7
  at_bf16x8 fq[KS][PARTS];
  const int own = row0 + wr * 16 + col;
  const bool live = own < rows;
  const int token = live ? own / a.group : 0, head = h * a.group + (live ? own - token * a.group : 0);
  const int64_t q_at = (s.first + token) * a.q_token + head * a.q_head + 8 * g;
  auto load_q = [&](int64_t at, bool there) {
#pragma unroll
    for (int ks = 0; ks < KS; ks++) query_parts<F32>(a.q, at + 32 * ks, there && 32 * ks + 8 * g < a.D, fq[ks]);
  };
  load_q(q_at, live);
#pragma unroll
  for (int ks = 0; ks < KS; ks++)
#pragma unroll
    for (int p = 0; p < PARTS; p++) asm volatile("" : "+v"(fq[ks][p]));  // (here from now on: a wait for it in the loop would be one for the next tile's loads)

  at_f32x4 acc[DT] = {};
  float m = -INFINITY, l = 0.f;  // the maximum so far times c; the sum of this lane's keys
  const bool busy = row0 + wr * 16 < rows;  // (a wave without rows loads with the others and leaves its SIMD to them)
  auto work = [&](int k0, auto last_, auto half) {
    constexpr bool last = decltype(last_)::value;  // the tile may have keys behind the last
#pragma unroll
    for (int u = 0; u < P::SUB; u++) {
      const int base = (u * WK + wk) * 32, key0 = k0 + base;
      if (last && key0 >= k_end) break;
      at_f32x4 sa = {0.f, 0.f, 0.f, 0.f}, sb = {0.f, 0.f, 0.f, 0.f};
      const int ra = half * KT + base + 8 * (col >> 2) + (col & 3), x = P::swz(ra);
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const int at = ra * DP + ((4 * ks + g) ^ x) * 8;
        const at_bf16x8 ka = frag(*reinterpret_cast<const u32x4*>(s_k + at)), kb = frag(*reinterpret_cast<const u32x4*>(s_k + at + 4 * DP));
#pragma unroll
        for (int p = PARTS - 1; p >= 0; p--) {  // the smallest part first
          sa = mma(ka, fq[ks][p], sa);
          sb = mma(kb, fq[ks][p], sb);
        }
      }
      at_bf16x8 fp[PARTS];
      float y[8], top;
      auto scores = [&](const at_f32x4& a0, const at_f32x4& b0) {
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = a0[j], y[4 + j] = b0[j];
        if (last) {
          const int left = k_end - key0 - 8 * g;
#pragma unroll
          for (int j = 0; j < 8; j++) y[j] = j < left ? y[j] : -INFINITY;
        }
        top = larger(larger(larger(y[0], y[1]), larger(y[2], y[3])), larger(larger(y[4], y[5]), larger(y[6], y[7])));
        top = across<16>(top);
        top = across<32>(top) * a.c;
      };
      scores(sa, sb);
      if (__ballot(F32 ? !(top <= m + 8.f) : top > m + 8.f)) {  // (weights of up to 2^8 do as well: most steps leave O alone)
        if constexpr (F32) {
          // An infinite element of a key makes a NaN with the second and third part of a query's, which may be 0: it counts with the first alone, which
          // has the sign.  Such scores, and those that are NaN anyway, are formed once more.
          if (__builtin_expect(__ballot(top != top) != 0, 0)) {
            at_f32x4 ta = {0.f, 0.f, 0.f, 0.f}, tb = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
              const int at = ra * DP + ((4 * ks + g) ^ x) * 8;
              const u32x4 ka = *reinterpret_cast<const u32x4*>(s_k + at), kb = *reinterpret_cast<const u32x4*>(s_k + at + 4 * DP);
              const at_bf16x8 fa = frag(u32x4{finite_pair(ka.x), finite_pair(ka.y), finite_pair(ka.z), finite_pair(ka.w)}),
                              fb = frag(u32x4{finite_pair(kb.x), finite_pair(kb.y), finite_pair(kb.z), finite_pair(kb.w)});
#pragma unroll
              for (int p = PARTS - 1; p > 0; p--) {
                ta = mma(fa, fq[ks][p], ta);
                tb = mma(fb, fq[ks][p], tb);
              }
              ta = mma(frag(ka), fq[ks][0], ta);
              tb = mma(frag(kb), fq[ks][0], tb);
            }
            scores(ta, tb);
          }
        }
        const float next = fmaxf(m, top), fix = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - next);
        m = next;
        l *= fix;
#pragma unroll
        for (int d = 0; d < DT; d++) acc[d] *= fix;
      }
      const float ref = m == -INFINITY ? 0.f : m;  // (nothing seen yet: every p is exp2(-inf))
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = __builtin_amdgcn_exp2f(fmaf(y[j], a.c, -ref));
      l += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
      if constexpr (!F32) {
        fp[0] = frag(u32x4{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7])});
      } else {
        uint32_t part[3][4];
#pragma unroll
        for (int j = 0; j < 4; j++) split2(y[2 * j], y[2 * j + 1], part[0][j], part[1][j], part[2][j]);
#pragma unroll
        for (int p = 0; p < 3; p++) fp[p] = frag(u32x4{part[p][0], part[p][1], part[p][2], part[p][3]});
      }
      // V^T: lane i of 16 asks for elements 4 (i % 4) .. + 3 of key 8 g + i / 4 and gets element i of keys 8 g .. + 3
      const int rv0 = half * KT + base + 8 * g + (col >> 2), xv = P::swz(rv0);
#pragma unroll
      for (int d = 0; d < DT; d++) {
        const int at = rv0 * DP + ((2 * d + ((col & 3) >> 1)) ^ xv) * 8 + (col & 1) * 4;
        typedef __attribute__((address_space(3))) at_s16x4* lds_ptr;
        const at_s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(s_v + at));
        const at_s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(s_v + at + 4 * DP));
        const at_bf16x8 fv = frag(__builtin_bit_cast(u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7)));
#pragma unroll
        for (int p = PARTS - 1; p >= 0; p--) acc[d] = mma(fv, fp[p], acc[d]);
      }
    }
  };
  typedef std::integral_constant<int, 0> Lower;
  typedef std::integral_constant<int, 1> Upper;
  int k0 = k_begin;  // the tile that is worked on
  if (k_begin < k_end) {
    put_tile(Lower());
    if (!ONE && k_begin + KT < k_end) ask_tile(k_begin + KT);
    __syncthreads();
  }
  if constexpr (ONE) {
    if (busy && k0 < k_end) work(k0, std::true_type(), Lower());
    // More keys than the host said: a tile at a time.  Where it lies and the rows of Q are found once more: they would else stay in registers, which costs most of what this form gains.
    for (k0 += KT; k0 < k_end; k0 += KT) {
      int t = tid;
      asm volatile("" : "+v"(t));
      __syncthreads();
#pragma unroll 1
      for (int e = t; e < KT * C; e += 256) {
        const int r = e / C, p = e % C, there = r * DP + (p ^ P::swz(r)) * 8;
        if (p >= real) continue;
        const bool good = k0 + r < k_end;
        *reinterpret_cast<u32x4*>(s_k + there) = *reinterpret_cast<global_row>(good ? k_at + (uint64_t)(k0 + r) * a.k_bytes + p * 16 : zero);
        *reinterpret_cast<u32x4*>(s_v + there) = *reinterpret_cast<global_row>(good ? v_at + (uint64_t)(k0 + r) * a.v_bytes + p * 16 : zero);
      }
      __syncthreads();
      const int row = row0 + wr * 16 + (t & 15);
      const bool has_row = row < rows;
      const int of = has_row ? row / a.group : 0;
      load_q((s.first + of) * a.q_token + (h * a.group + (has_row ? row - of * a.group : 0)) * a.q_head + 8 * (t >> 4 & 3), has_row);
      if (busy) work(k0, std::true_type(), Lower());
    }
  } else {
    auto turn = [&](auto last_, auto half, auto other) {
      if (busy) work(k0, last_, half);
      k0 += KT;
      if (k0 < k_end) {  // into the other half of LDS: everyone is past the tile that was there
        put_tile(other);
        if (k0 + KT < k_end) ask_tile(k0 + KT);
        __syncthreads();
      }
    };
    // Whole tiles in turns whose halves of LDS are constants; then, in code of its own, the one that may end before its last key.
    int half = 0;
    while (k0 + KT <= k_end) {
      turn(std::false_type(), Lower(), Upper());
      half = 1;
      if (k0 + KT > k_end) break;
      turn(std::false_type(), Upper(), Lower());
      half = 0;
    }
    if (k0 < k_end) turn(std::true_type(), half, half ^ 1);
  }
  l = sum32(sum16(l));

  auto put = [&](int row, int d, at_f32x4 x, float mm, float sum) {
    cross_put<F32>(a, place, row, row / a.group, h * a.group + row % a.group, d, x, mm, sum);
  };
  if constexpr (WK == 1) {
    if (!live) return;
#pragma unroll
    for (int d = 0; d < DT; d++) put(own, 16 * d + 4 * g, acc[d], m, l);
  } else {
    // The waves along keys meet in LDS: O of a row where the keys were, its maximum and sum where the values were.
    constexpr int Q4 = DT * 4, IT = (16 * Q4 + WK * 64 - 1) / (WK * 64);  // quads of a row; quads of a lane
    float* so = reinterpret_cast<float*>(s_k);            // [wave][16][DT * 16]
    float* sm = reinterpret_cast<float*>(s_v);            // [wave][16][2]
    static_assert(4 * 16 * DT * 16 * 4 <= 2 * KT * DP * 2, "");
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; d++) *reinterpret_cast<at_f32x4*>(so + ((wave * 16 + col) * Q4 + ((4 * d + g) ^ (col & 3))) * 4) = acc[d];
    if (g == 0) {
      sm[(wave * 16 + col) * 2] = m;
      sm[(wave * 16 + col) * 2 + 1] = l;
    }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < IT; it++) {
      const int e = wk * 64 + lane + it * WK * 64, r = e / Q4, p = e % Q4;
      const int row = row0 + wr * 16 + r;
      if (r >= 16 || row >= rows) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WK; w++) top = fmaxf(top, sm[((w * WR + wr) * 16 + r) * 2]);
      const float ref = top == -INFINITY ? 0.f : top;
      at_f32x4 x = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < WK; w++) {
        const int at = (w * WR + wr) * 16 + r;
        const float f = __builtin_amdgcn_exp2f(sm[at * 2] - ref);
        sum += sm[at * 2 + 1] * f;
        x += *reinterpret_cast<const at_f32x4*>(so + (at * Q4 + (p ^ (r & 3))) * 4) * f;
      }
      put(row, p * 4, x, top, sum);
    }
  }
}

// Many rows of bf16 queries: a wave has 32 NR of them, v_mfma_f32_32x32x16_bf16, DK steps of 16 elements in the first product and DT tiles of 32 in the second.  First operand rows
// 8 a + 4 b + c = keys 16 (a / 2) + 8 b + 4 (a % 2) + c leave a lane with one row of Q and, of every 16 keys, the eight consecutive ones that the second product takes.
// Keys and values go from memory to LDS directly.  FULL: heads of 16 DK elements.
template <int DK, int DT>
struct Wide {
  static constexpr int C = DK == 5 ? 12 : 2 * DK, DP = 8 * C, KT = 64;  // (pieces of a row in LDS: ten of them would lie in the same banks every third row)
  static constexpr int CHUNKS = KT * C / 64;                            // 64 pieces each, a wave's load
  static constexpr bool ONES = DK == 5;                                 // the tiles of 32 of the second product reach behind the values: what lies there is 1, and O has the sum of the weights
  // Eight lanes of a key operand have rows 0 - 3 and 8 - 11 (or 4 - 7 and 12 - 15) and one piece, 32 of a value operand four rows and the four pieces of a tile of 32: each in banks of their own.
  // A KB of values, pitch 10 / 12 / 16 / 16 pieces with rows exclusive-ored by 0 / row / 4 / row / 0 / 4 (row % 4): 3.4 / 2.0 / 6.8 / 1.9 ns.
  static __device__ __forceinline__ int swz(int row) {
    return C == 16 ? (row & 3) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1) : C == 12 ? (row >> 2) & 3 : ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
  }
};
typedef float at_f32x16 __attribute__((ext_vector_type(16)));
// the sum of two bf16 and z
__device__ __forceinline__ float pair_sum(uint32_t w, float z) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3f803f80u), z, false);
}
__device__ __forceinline__ at_f32x16 mma32(at_bf16x8 x, at_bf16x8 y, at_f32x16 acc) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, acc, 0, 0, 0); }

template <int DK, int DT, int NR, bool FULL>
__global__ __launch_bounds__(256, DK <= 6 && NR == 1 ? 3 : 2) void cross_wide_kernel(CrossArgs a) {
  typedef Wide<DK, DT> P;
  constexpr int KT = P::KT, C = P::C, DP = P::DP, CHUNKS = P::CHUNKS;
  __shared__ __align__(16) uint16_t s_all[4 * KT * DP];
  // in LDS: two tiles of values, two of keys
  constexpr int TILE = KT * DP;
  // Of three or four waves of a SIMD the ones that multiply go first, and the others' exponents fill what they leave: heads of 64, 3000 tokens 65.6 -> 59.2 us, 200 over 2000 keys 36.6 -> 34.1, heads of
  // 80 76.8 -> 72.5.  (Of two waves, heads of 128, 3 x 700 tokens over up to 6404 keys 179 -> 190: the compiler moves nothing over the switches.)
  constexpr bool URGENT = DK <= 5 && NR == 1;
  CrossPlace place;
  if (!cross_place(a, place)) return;
  const CrossSeq& s = place.s;
  const int h = place.h, rows = place.rows, row0 = place.row0, k_begin = place.k_begin, k_end = place.k_end;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, g = lane >> 5;

  // Two waves load keys and two values, half of a tile each: chunks of 64 pieces one behind the other in LDS, of which a lane loads the one that swz puts there.  Pieces behind a head's
  // end are zeros (ones, where O has the sum) from the beginning.
  constexpr int NLOAD = CHUNKS / 2;
  const bool keys = wave < 2;
  const int real = a.D / 8;
  const uint32_t bytes = keys ? a.k_bytes : a.v_bytes;
  const uint64_t base = (uint64_t)(uintptr_t)(keys ? a.k + h * a.k_head : a.v + h * a.v_head) + s.key * bytes;
  uint16_t* const to = s_all + (keys ? 2 * TILE : 0) + (wave & 1) * (TILE / 2);
  uint32_t off[NLOAD];
#pragma unroll
  for (int i = 0; i < NLOAD; i++) {
    const int e = ((wave & 1) * NLOAD + i) * 64 + lane, r = e / C, p = (e % C) ^ P::swz(r);
    off[i] = p < real ? r * bytes + p * 16 : ~0u;
    if (!FULL && p >= real) {
      const uint32_t fill = P::ONES && !keys && p >= 2 * DK ? 0x3f803f80u : 0;
#pragma unroll
      for (int t = 0; t < 2; t++) *reinterpret_cast<u32x4*>(to + t * TILE + (i * 64 + lane) * 8) = u32x4{fill, fill, fill, fill};
    }
  }
  typedef const __attribute__((address_space(1))) char* global_ptr;
  typedef const __attribute__((address_space(1))) void* global_any;
  typedef __attribute__((address_space(3))) void* lds_ptr;
  auto ask = [&](int k0, int half) {
    if (k0 >= k_end) return;
    const global_ptr at = reinterpret_cast<global_ptr>(base + (uint64_t)k0 * bytes);
    if (k0 + KT <= k_end) {
#pragma unroll
      for (int i = 0; i < NLOAD; i++)
        if (FULL || off[i] != ~0u) __builtin_amdgcn_global_load_lds((global_any)(at + off[i]), (lds_ptr)(to + half * TILE + i * 512), 16, 0, 0);
      return;
    }
#pragma unroll
    for (int i = 0; i < NLOAD; i++) {  // (keys behind the last: zeros)
      const int r = (((wave & 1) * NLOAD + i) * 64 + lane) / C;
      const global_ptr from = k0 + r < k_end ? at + off[i] : reinterpret_cast<global_ptr>((uint64_t)(uintptr_t)g_no_state);
      if (FULL || off[i] != ~0u) __builtin_amdgcn_global_load_lds((global_any)from, (lds_ptr)(to + half * TILE + i * 512), 16, 0, 0);
    }
  };
  // Q: second operand, row `col`, elements 16 s + 8 g .. + 7
  at_bf16x8 fq[NR][DK];
  int row[NR], token[NR], head[NR];
  bool live[NR];
#pragma unroll
  for (int r = 0; r < NR; r++) {
    row[r] = row0 + (wave * NR + r) * 32 + col;
    live[r] = row[r] < rows;
    token[r] = live[r] ? row[r] / a.group : 0;
    head[r] = h * a.group + (live[r] ? row[r] - token[r] * a.group : 0);
    at_bf16x8 part[1];
#pragma unroll
    for (int ks = 0; ks < DK; ks++) {
      query_parts<false>(a.q, (s.first + token[r]) * a.q_token + head[r] * a.q_head + 16 * ks + 8 * g, live[r] && 16 * ks + 8 * g < a.D, part);
      fq[r][ks] = part[0];
    }
  }
  at_f32x16 acc[NR][DT] = {};
  float m[NR], l2[NR][2] = {};  // the maximum so far times c; the sums of this lane's keys
#pragma unroll
  for (int r = 0; r < NR; r++) m[r] = -INFINITY;
  const int krow = (col & 3) | ((col >> 3) & 1) << 2 | ((col >> 2) & 1) << 3 | (col >> 4) << 4;
  auto arrived = [&]() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  auto turn = [&](int k0, auto last_, int half) {
    constexpr bool last = decltype(last_)::value;
    const uint16_t *v = s_all + half * TILE, *k = v + 2 * TILE;
    arrived();
    if (!last) ask(k0 + KT, half ^ 1);
#pragma unroll
    for (int u = 0; u < 2; u++) {
      if (last && k0 + 32 * u >= k_end) break;
      at_f32x16 ys[NR] = {};
      {
        const int r = u * 32 + krow, x = P::swz(r);
        if (URGENT) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < DK; ks++) {
          const at_bf16x8 fk = frag(*reinterpret_cast<const u32x4*>(k + r * DP + ((2 * ks + g) ^ x) * 8));
#pragma unroll
          for (int n = 0; n < NR; n++) ys[n] = mma32(fk, fq[n][ks], ys[n]);
        }
      }
      if (URGENT) __builtin_amdgcn_s_setprio(0);
      at_bf16x8 fp[NR][2];
#pragma unroll
      for (int n = 0; n < NR; n++) {
        at_f32x16& y = ys[n];
        if (last) {
          const int left = k_end - k0 - 32 * u - 8 * g;
#pragma unroll
          for (int j = 0; j < 16; j++) y[j] = 16 * (j >> 3) + (j & 7) < left ? y[j] : -INFINITY;
        }
        float top = larger(larger(y[0], y[1]), y[2]);
#pragma unroll
        for (int j = 3; j < 15; j += 2) top = larger(larger(y[j], y[j + 1]), top);
        top = larger(top, y[15]);
        top = across<32>(top) * a.c;
        if (__ballot(top > m[n] + 8.f)) {  // (weights of up to 2^8 do as well: most tiles leave O alone)
          const float next = fmaxf(m[n], top), fix = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - next);
          m[n] = next;
          l2[n][0] *= fix;
          l2[n][1] *= fix;
#pragma unroll
          for (int d = 0; d < DT; d++) acc[n][d] *= fix;
        }
        const float ref = m[n] == -INFINITY ? 0.f : m[n];  // (nothing seen yet: every p is exp2(-inf))
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
          float e[8];
#pragma unroll
          for (int j = 0; j < 8; j++) e[j] = __builtin_amdgcn_exp2f(fmaf(y[8 * hf + j], a.c, -ref));
          const u32x4 w = {pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]), pack_bf16(e[4], e[5]), pack_bf16(e[6], e[7])};
          fp[n][hf] = frag(w);
          if (!P::ONES) {  // (the sum of the weights as they are multiplied, two an instruction)
            l2[n][hf] = pair_sum(w.x, pair_sum(w.y, l2[n][hf]));
            l2[n][hf] = pair_sum(w.z, pair_sum(w.w, l2[n][hf]));
          }
        }
      }
      if (URGENT) __builtin_amdgcn_s_setprio(1);
      // V^T: lane i of 16 asks for elements 4 (i % 4) .. + 3 of key 8 g + i / 4 and gets element i of keys 8 g .. + 3
      const int i = lane & 15, upper = (lane >> 4) & 1;
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        const int r = 32 * u + 16 * kk + 8 * g + (i >> 2), x = P::swz(r), x4 = P::swz(r + 4);
#pragma unroll
        for (int d = 0; d < DT; d++) {
          const int p = 4 * d + 2 * upper + ((i & 3) >> 1);
          typedef __attribute__((address_space(3))) at_s16x4* lds_quad;
          const at_s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)(v + r * DP + (p ^ x) * 8 + (i & 1) * 4));
          const at_s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)(v + (r + 4) * DP + (p ^ x4) * 8 + (i & 1) * 4));
          const at_bf16x8 fv = frag(__builtin_bit_cast(u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7)));
#pragma unroll
          for (int n = 0; n < NR; n++) acc[n][d] = mma32(fv, fp[n][kk], acc[n][d]);
        }
      }
    }
  };
  ask(k_begin, 0);
  int k0 = k_begin, half = 0;
  for (; k0 + KT < k_end; k0 += KT, half ^= 1) turn(k0, std::false_type(), half);
  if (k0 < k_end) turn(k0, std::true_type(), half);
#pragma unroll
  for (int n = 0; n < NR; n++) {
    const float l = P::ONES ? acc[n][DT - 1][8] : sum32(l2[n][0] + l2[n][1]);  // (element 16 DK of O, and four behind it in the other half of the lanes)
    if (!live[n]) continue;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        cross_put<false>(a, place, row[n], token[n], head[n], 32 * d + 8 * j + 4 * g,
                         at_f32x4{acc[n][d][4 * j], acc[n][d][4 * j + 1], acc[n][d][4 * j + 2], acc[n][d][4 * j + 3]}, m[n], l);
  }
}

// Joins the pieces of a row: 16 bytes of it per lane, L lanes a row, G groups of lanes along the pieces
template <int L, bool F32, int G>
__global__ __launch_bounds__(256) void cross_join_kernel(CrossArgs a) {
  constexpr int PER = 256 / L / G;
  __shared__ at_f32x4 s_x[G > 1 ? 256 : 1];
  __shared__ float s_ml[G > 1 ? 256 / L * 2 : 1];
  const int tid = threadIdx.x, d = tid % L * 4, tile = blockIdx.y;
  int place, rt;
  cross_tile(a, a.whole + tile, place, rt);
  const int b = place / a.kv, h = place % a.kv;
  const CrossSeq s = cross_sequence(a, b);
  int per, pieces;
  cut(a, s.keys, per, pieces);
  const int i = blockIdx.x * PER + tid / L % PER, group = tid / L / PER, row = rt * a.rows_of_tile + i;
  if (pieces < 2) return;
  const bool live = i < a.rows_of_tile && row < s.n * a.group && d < a.D;
  const int64_t all = (int64_t)(a.tiles - a.whole) * a.rows_of_tile, at = (int64_t)tile * a.rows_of_tile + i;
  float m = -INFINITY, sum = 0.f;
  at_f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    constexpr int U = 4;
    for (int k = group; k < pieces; k += U * G) {
      float mk[U], lk[U];
      at_f32x4 xk[U];
#pragma unroll
      for (int j = 0; j < U; j++) {
        const int64_t from = min(k + j * G, pieces - 1) * all + at;
        mk[j] = a.part_ml[2 * from];
        lk[j] = a.part_ml[2 * from + 1];
        xk[j] = *reinterpret_cast<const at_f32x4*>(a.part_o + from * a.D + d);
      }
#pragma unroll
      for (int j = 0; j < U; j++) {
        if (k + j * G >= pieces) break;
        const float next = fmaxf(m, mk[j]), ref = next == -INFINITY ? 0.f : next;
        const float f = __builtin_amdgcn_exp2f(m - ref), fk = __builtin_amdgcn_exp2f(mk[j] - ref);
        x = x * f + xk[j] * fk;
        sum = sum * f + lk[j] * fk;
        m = next;
      }
    }
  }
  if constexpr (G > 1) {
    s_x[tid] = x;
    if (d == 0) {
      s_ml[tid / L * 2] = m;
      s_ml[tid / L * 2 + 1] = sum;
    }
    __syncthreads();
    if (group) return;
    float top = -INFINITY;
    for (int k = 0; k < G; k++) top = fmaxf(top, s_ml[(k * PER + tid / L) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
    x = at_f32x4{0.f, 0.f, 0.f, 0.f};
    sum = 0.f;
    for (int k = 0; k < G; k++) {
      const float f = __builtin_amdgcn_exp2f(s_ml[(k * PER + tid / L) * 2] - ref);
      x += s_x[tid + k * PER * L] * f;
      sum += s_ml[(k * PER + tid / L) * 2 + 1] * f;
    }
  }
  if (!live) return;
  x *= sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
  const int t = row / a.group;
  const int64_t to = (s.first + t) * a.o_token + (h * a.group + row - t * a.group) * a.o_head + d;
  if (F32) *reinterpret_cast<at_f32x4*>(reinterpret_cast<float*>(a.o) + to) = x;
  else *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(a.o) + to) = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
}

// ---- host side ------------------------------------------------------------------------------------------------------------
struct CrossPlan {
  int nq, wr, row_tiles, rows_of_tile, pieces, min_tiles;
  int64_t whole, tiles;
  bool one;  // tile of keys a sequence
};
// Rows of a wave by the rows there are: 16, 32, and 64 where heads are of 96 elements at most, there is work for all CUs and the last tile's idle rows weigh little (each row of LDS read is
// used twice, a SIMD has two waves instead of three or four.  Heads of 80, 64 / 32 rows: 16 heads, 7000 tokens 302 / 348 us, 64 sequences of 200 tokens 32.1 / 39.1; but 8 of 1100
// 71.8 / 67.4, and with few tiles 2 of 600 over 6000 keys 93 / 67).  CUs have two workgroups each (one, of 64 rows a wave: 4900 tokens over 4900 keys 176 us, with two 209): as many
// row tiles as make whole rounds go through all of their keys, the keys of those that are left are cut into as many pieces as fill another, of two tiles and of twice as many keys as rows at least.
// Few keys are not cut, for the second launch takes longer than they do: two tokens of 32 heads of 128 over 179 keys 9.8 us cut, 7.1 uncut, over 300 10.1 both, over 500 10.6 and 12.3; heads of 64 over 300 9.6 and 7.8, over
// 500 9.7 and 12.0.
static CrossPlan cross_plan(bool f32, int64_t B, int heads, int kv, int64_t max_tokens, int64_t max_keys, int D) {
  CrossPlan p;
  if (max_keys > 0x7fffffff) max_keys = 0x7fffffff;
  const int64_t rows = max_tokens * (heads / kv);
  const int64_t narrow = (rows + 127) / 128, twice = (narrow + 1) / 2;
  p.nq = rows <= 64 || f32 || D > 128 || max_keys <= 64 ? 1 : D > 96 || twice * B * kv < 384 || (narrow % 2 && narrow < 20) ? 2 : 4;
  p.wr = rows <= 32 ? 2 : 4;
  p.one = max_keys <= 64;
  p.rows_of_tile = p.nq * 16 * p.wr;
  const int64_t per = p.rows_of_tile, row_tiles = (rows + per - 1) / per;
  p.row_tiles = (int)row_tiles;
  const int64_t least = (2 * (rows < per ? rows : per) + 63) / 64;
  p.min_tiles = (int)(least > 2 ? least : 2);
  const int64_t slots = p.nq == 4 ? 256 : 512, most = (max_keys + p.min_tiles * 64 - 1) / (p.min_tiles * 64);
  p.tiles = B * kv * row_tiles;
  p.whole = p.tiles / slots * slots;
  const int64_t rest = p.tiles - p.whole, wanted = rest ? slots / rest : 1;
  p.pieces = (int)(max_keys <= (D <= 64 ? 384 : 256) || most < 2 || wanted < 2 ? 1 : wanted < most ? wanted : most);
  if (p.pieces == 1) p.whole = p.tiles;
  return p;
}
static size_t cross_room(const CrossPlan& p, int D) { return (size_t)(p.tiles - p.whole) * p.pieces * p.rows_of_tile * (D + 2) * sizeof(float); }
// Elements of a head that are held, tiles of 16 and steps of 16 they take (the latter of the forms with products of 32 x 32)
template <int DP, int DT, int DK>
static void cross_launch(const CrossPlan& p, bool f32, dim3 grid, hipStream_t st, const CrossArgs& a) {
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, a); };
  if constexpr (DK > 0) {
    if (p.nq == 1 && p.wr == 4 && p.one) return f32 ? go(cross_kernel<DP, DT, 4, true, true>) : go(cross_kernel<DP, DT, 4, false, true>);
  }
  if (f32) return p.wr == 2 ? go(cross_kernel<DP, DT, 2, true, false>) : go(cross_kernel<DP, DT, 4, true, false>);
  if (p.nq == 1) return p.wr == 2 ? go(cross_kernel<DP, DT, 2, false, false>) : go(cross_kernel<DP, DT, 4, false, false>);
  if constexpr (DK > 0) {
    constexpr int D2 = (DK + 1) / 2;
    const bool full = a.D == 16 * DK;
    if constexpr (DK <= 6) {
      if constexpr (DK != 5) {
        if (p.nq == 4 && full) return go(cross_wide_kernel<DK, D2, 2, true>);
      }
      if (p.nq == 4) return go(cross_wide_kernel<DK, D2, 2, false>);
    }
    if constexpr (DK != 5) {
      if (full) return go(cross_wide_kernel<DK, D2, 1, true>);
    }
    go(cross_wide_kernel<DK, D2, 1, false>);
  }
}
static bool cross_sizes(int dtype, int64_t T, int64_t B, int heads, int kv, int head_dim, int64_t max_tokens, int64_t max_keys) {
  return (dtype == MLLM_HIP_F32 || dtype == MLLM_HIP_BF16) && T >= 0 && B >= 0 && heads >= 1 && kv >= 1 && head_dim >= 1 && max_tokens >= 0 && max_keys >= 0;
}
static bool cross_shape(int64_t T, int64_t B, int heads, int kv, int head_dim, int64_t max_tokens) {
  return head_dim % 8 == 0 && head_dim <= 256 && heads % kv == 0 && heads <= 65536 && T <= 0x7fff0000 / heads && B <= 0x7fffffff / heads && max_tokens <= 0x7fffffff / heads;
}

}  // namespace mllmhip

using namespace mllmhip;

MLLM_API size_t mllm_hip_attention_cross_workspace_bytes(int dtype, int64_t T, int64_t B, int heads, int kv_heads, int head_dim, int64_t max_tokens, int64_t max_keys) {
  if (!cross_sizes(dtype, T, B, heads, kv_heads, head_dim, max_tokens, max_keys) || !cross_shape(T, B, heads, kv_heads, head_dim, max_tokens)) return 0;
  if (T == 0 || B == 0 || max_tokens == 0) return 0;
  if (max_tokens > T) max_tokens = T;
  return cross_room(cross_plan(dtype == MLLM_HIP_F32, B, heads, kv_heads, max_tokens, max_keys, head_dim), head_dim);
}

MLLM_API int mllm_hip_attention_cross(const mllm_hip_heads* q, int dtype, int64_t T, const mllm_hip_states* kv, const int32_t* cu_tokens, const int32_t* key_first,
                                      const int32_t* key_count, int64_t B, int64_t max_tokens, int64_t max_keys, float scale, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  if (!q || !kv || kv->keys < 0 || !(scale > 0.f) || scale > 2e38f) return MLLM_HIP_E_BADARG;
  if (!cross_sizes(dtype, T, B, q->heads, kv->heads, kv->head_dim, max_tokens, max_keys)) return MLLM_HIP_E_BADARG;
  if (!cross_shape(T, B, q->heads, kv->heads, kv->head_dim, max_tokens) || kv->keys > 0x40000000 || kv->k_stride < 0 || kv->v_stride < 0 || kv->k_stride > (1 << 23) ||
      kv->v_stride > (1 << 23))  // (the kernels' places of keys go tiles past the last)
    return MLLM_HIP_E_SHAPE;
  if (T == 0 || B == 0 || max_tokens == 0) return 0;
  if (max_tokens > T) max_tokens = T;
  if (!q->x || !q->y || (kv->keys && (!kv->k || !kv->v)) || !cu_tokens || !key_first || !key_count) return MLLM_HIP_E_BADARG;
  const int wide = dtype == MLLM_HIP_F32 ? 4 : 2;
  auto al = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  auto whole = [&](int64_t stride) { return stride * wide % 16 == 0; };
  if (!al(q->x, 16) || !al(q->y, 16) || !al(kv->k, 16) || !al(kv->v, 16) || !whole(q->x_token_stride) || !whole(q->x_head_stride) || !whole(q->y_token_stride) ||
      !whole(q->y_head_stride) || kv->k_stride % 8 || kv->v_stride % 8 || kv->k_head_stride % 8 || kv->v_head_stride % 8 || !al(cu_tokens, 4) || !al(key_first, 4) ||
      !al(key_count, 4) || !al(workspace, 16))
    return MLLM_HIP_E_ALIGN;
  if (q->x == q->y || !own_places(*q, T)) return MLLM_HIP_E_BADARG;
  const bool f32 = dtype == MLLM_HIP_F32;
  const int heads = q->heads, D = kv->head_dim;
  const CrossPlan p = cross_plan(f32, B, heads, kv->heads, max_tokens, max_keys, D);
  const size_t need = cross_room(p, D);
  if (need && (!workspace || workspace_bytes < need)) return MLLM_HIP_E_BADARG;
  if (p.whole + (p.tiles - p.whole) * p.pieces > 0xffffff) return MLLM_HIP_E_SHAPE;
  CrossArgs a = {};
  a.q = q->x;
  a.o = q->y;
  a.q_token = q->x_token_stride;
  a.q_head = q->x_head_stride;
  a.o_token = q->y_token_stride;
  a.o_head = q->y_head_stride;
  a.k = reinterpret_cast<const uint16_t*>(kv->k);
  a.v = reinterpret_cast<const uint16_t*>(kv->v);
  a.k_head = kv->k_head_stride;
  a.v_head = kv->v_head_stride;
  a.k_bytes = (uint32_t)kv->k_stride * 2;
  a.v_bytes = (uint32_t)kv->v_stride * 2;
  a.cu = cu_tokens;
  a.first = key_first;
  a.count = key_count;
  a.keys = kv->keys;
  a.T = (int)T;
  a.B = (int)B;
  a.kv = kv->heads;
  a.group = heads / kv->heads;
  a.D = D;
  a.max_tokens = (int)max_tokens;
  a.row_tiles = p.row_tiles;
  a.rows_of_tile = p.rows_of_tile;
  a.pieces = p.pieces;
  a.min_tiles = p.min_tiles;
  a.whole = (int)p.whole;
  a.tiles = (int)p.tiles;
  a.c = scale * 1.44269504088896341f;
  a.part_o = reinterpret_cast<float*>(workspace);
  const int64_t rest = p.tiles - p.whole;
  a.part_ml = rest ? a.part_o + (size_t)rest * p.pieces * p.rows_of_tile * D : nullptr;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(p.whole + rest * p.pieces));
  if (D <= 64) cross_launch<64, 4, 4>(p, f32, grid, st, a);
  else if (D <= 80) cross_launch<96, 5, 5>(p, f32, grid, st, a);
  else if (D <= 96) cross_launch<96, 6, 6>(p, f32, grid, st, a);
  else if (D <= 128) cross_launch<128, 8, 8>(p, f32, grid, st, a);
  else cross_launch<256, 16, 0>(p, f32, grid, st, a);
  RC_RET((int)hipGetLastError());
  if (rest) {
    const bool many = p.pieces >= 8;  // lanes along the pieces
    const int lanes = D <= 64 ? 16 : D <= 128 ? 32 : 64, per = many ? 1 : 256 / lanes;
    const int64_t rows = max_tokens * a.group, most = rows < p.rows_of_tile ? rows : p.rows_of_tile;
    const dim3 jgrid((unsigned)((most + per - 1) / per), (unsigned)rest);
    auto join = [&](auto kern) { hipLaunchKernelGGL(kern, jgrid, dim3(256), 0, st, a); };
#define JOIN(L_)                                                              \
  if (many) {                                                                 \
    if (f32) join(cross_join_kernel<L_, true, 256 / L_>);                     \
    else join(cross_join_kernel<L_, false, 256 / L_>);                        \
  } else {                                                                    \
    if (f32) join(cross_join_kernel<L_, true, 1>);                            \
    else join(cross_join_kernel<L_, false, 1>);                               \
  }
    if (lanes == 16) { JOIN(16) }
    else if (lanes == 32) { JOIN(32) }
    else { JOIN(64) }
#undef JOIN
  }
  return (int)hipGetLastError();
}
