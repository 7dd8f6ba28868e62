// A token from every row of logits by temperature, top-k, top-p, min-p and a given uniform number, for gfx950.
//
//   w_i = exp((x_i - max) / t), below 2^-52: 0.  In descending order (equal logits: lowest index first) the first k are kept, of these the
//   shortest beginning whose mass is p of theirs or more, of these the ones with w >= min_p.  The token is the first kept one, in the order of
//   the vocabulary, at which the running sum of the weights exceeds u times their sum.
//
// Nothing is sorted: what is kept is everything above a border (a logit and how many of its equals), and the border is found by counts and masses.
// A row is cut into pieces, a workgroup each, and goes through four launches that meet in the workspace:
//   1  maximum and minimum of every piece
//   2  counts and masses over 512 equal steps from the row's maximum down to where weights vanish
//   3  the step (or steps) the border lies in; sums of the weights above it, piece by piece; the elements within it, in order of their index
//   4  one workgroup per row: the border itself, by counts and masses over ever narrower ranges of the bits of those elements' logits; the piece
//      in which the running sum crosses u, and the element
// The row is read three times, from memory once (a row of 151 936 stays in the caches).  Weights and their sums are fp64; the masses that
// find the border are added by atomics and therefore integers, in units of 2^-44 at 151 936 logits: sums that do not depend on an order.
#include "item8.h"

namespace mllmhip {

enum { SMP_STEPS = 512, SMP_WG = 512, SMP_BINS = 2048, SMP_LAST = 1024, SMP_RANKED = 512, SMP_PIECES = 16 };

struct SampleRow {  // what launch 3 finds out about a row
  int lo, hi;       // the border's steps; lo = SMP_STEPS: everything is kept
  int cut;          // 1: the k-th is within the row's weights
  uint32_t above;   // elements in front of step lo
  uint64_t mass_above, mass;  // of the elements in front of step lo, of all (both in units)
  uint32_t listed;
  int pad;
};
struct SampleArgs {
  const void* x;
  int64_t stride;
  int rows, V, pieces;
  const float *u, *t, *p, *min_p;
  const int32_t* k;
  int32_t* token;
  double unit;  // units of mass per weight of 1
  // workspace
  float* ends;      // [rows][pieces][2]: maximum, minimum
  int* top;         // [rows][pieces]: index of the maximum
  uint32_t* count;  // [rows][pieces][SMP_STEPS]
  uint64_t* mass;   // the same
  double* sum;      // [rows][pieces]
  uint32_t* from;   // [rows][pieces]: where the piece's elements begin in the list
  uint32_t* list;   // [rows][V]
  SampleRow* row;
};

template <int XT>
struct SampleVec {
  static constexpr int N = XT == MLLM_HIP_F32 ? 4 : 8;  // logits of 16 bytes
};
// a logit as the operator takes it: no number counts as -inf, -0 as 0
__device__ __forceinline__ float logit(float v) { return v != v ? -INFINITY : v + 0.0f; }
__device__ __forceinline__ uint32_t key_of(float v) {  // larger logits, larger keys
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// A row as 16-byte vectors: `head` elements in front of the first aligned one, `vecs` vectors, the rest behind.
template <int XT>
struct SampleSpan {
  static constexpr int N = SampleVec<XT>::N;
  const char* x;
  int V, head, vecs;
  __device__ __forceinline__ SampleSpan(const SampleArgs& a, int row) {
    constexpr int wide = 16 / N;
    x = reinterpret_cast<const char*>(a.x) + row * a.stride * wide;
    V = a.V;
    head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / wide);
    vecs = (V - head) / N;
  }
  __device__ __forceinline__ float at(int i) const {
    return logit(XT == MLLM_HIP_F32 ? reinterpret_cast<const float*>(x)[i] : bf16_to_f32(reinterpret_cast<const uint16_t*>(x)[i]));
  }
  // Calls f(i, v, n) in the order of the index for vectors v0 .. v1 - 1 by a wave, with the elements in front of the first and behind the last vector of
  // the row: a lane's n elements v[0 .. n - 1] are i .. i + n - 1 (lanes in ascending order; every lane comes along, with n = 0 if it has none)
  template <typename F>
  __device__ __forceinline__ void walk(int v0, int v1, F&& f) const {
    const int lane = threadIdx.x & 63;
    float v[N];
    if (v0 == 0 && head) {
      v[0] = lane < head ? at(lane) : 0.f;
      f(lane, v, lane < head ? 1 : 0);
    }
    constexpr int U = 4;  // vectors in flight
    for (int b = v0; b < v1; b += 64 * U) {
      u32x4 r[U];
#pragma unroll
      for (int j = 0; j < U; j++) {
        const int at_ = min(b + j * 64 + lane, v1 - 1);
        r[j] = *reinterpret_cast<const u32x4*>(x + (int64_t)head * (16 / N) + (int64_t)at_ * 16);
      }
#pragma unroll
      for (int j = 0; j < U; j++) {
        if (b + j * 64 >= v1) break;
        const int at_ = b + j * 64 + lane;
        const uint32_t w[4] = {r[j].x, r[j].y, r[j].z, r[j].w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (XT == MLLM_HIP_F32) {
            v[e] = logit(__uint_as_float(w[e]));
          } else {
            v[2 * e % N] = logit(__uint_as_float(w[e] << 16));
            v[(2 * e + 1) % N] = logit(__uint_as_float(w[e] & 0xffff0000u));
          }
        }
        f(head + at_ * N, v, at_ < v1 ? N : 0);
      }
    }
    const int tail = head + vecs * N;
    if (v1 == vecs && tail < V) {
      v[0] = tail + lane < V ? at(tail + lane) : 0.f;
      f(tail + lane, v, tail + lane < V ? 1 : 0);
    }
  }
};
// vectors of wave `wave` of `waves` in piece p
__device__ __forceinline__ void share(int vecs, int pieces, int p, int waves, int wave, int& v0, int& v1) {
  const int per = (vecs + pieces - 1) / pieces, a = min(vecs, p * per), b = min(vecs, a + per), each = (b - a + waves - 1) / waves;
  v0 = min(b, a + wave * each);
  v1 = min(b, v0 + each);
  // who has the row's first or last vector also has what is in front of or behind it; a row without vectors belongs to the first wave
  if (vecs == 0) v0 = 0, v1 = p == 0 && wave == 0 ? 0 : -1;
  else if (v0 == v1) v0 = v1 = -1;
}

// A row's weights: its maximum, what divides its logits, and the steps
struct SampleScale {
  float top, step;
  double c;       // 64 / (t ln 2)
  bool infinite;  // the maximum is: its equals weigh 1, the rest nothing
  float min_w;
  const double* table;  // 2^(j / 64), j = 0 .. 63
  // exp((v - top) / t) = 2^(n / 64) e^(r ln 2 / 64) with n + r = (v - top) c, |r| <= 1/2: the table, a power of two and five terms of the series (the
  // sixth is under 2^-54).  Off by 2^-52 and what rounding (v - top) c leaves of up to 36, 2^-47; the library's exp of a quotient took three times as long.
  __device__ __forceinline__ double weight(float v) const {
    if (infinite) return v == INFINITY ? 1.0 : 0.0;
    const double y = ((double)v - (double)top) * c;
    if (!(y > -3328.0)) return 0.0;  // 52 * 64: below 2^-52
    const double n = rint(y), r = (y - n) * 0.010830424696249145;
    const int i = (int)n;
    double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    e = fma(r, e, 1.0 / 6.0);
    e = fma(r, e, 0.5);
    e = fma(r, e, 1.0);
    e = fma(r, e, 1.0);
    return __builtin_ldexp(e * table[i & 63], i >> 6);
  }
  // the step of a logit; SMP_STEPS: its weight is below 2^-52
  __device__ __forceinline__ int step_of(float v) const {
    if (infinite) return v == INFINITY ? 0 : SMP_STEPS;
    const float q = (top - v) * step;
    return q < (float)SMP_STEPS ? (int)q : SMP_STEPS;
  }
  __device__ __forceinline__ bool heavy(double w) const { return w > 0.0 && w >= (double)min_w; }
};
// (the caller waits for the other waves before it takes a weight)
__device__ __forceinline__ SampleScale scale_of(const SampleArgs& a, int row, double* table) {
  SampleScale s;
  if (threadIdx.x < 64) table[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
  s.table = table;
  float top = -INFINITY, low = INFINITY;
  for (int i = threadIdx.x & 63; i < a.pieces; i += 64) {
    top = fmaxf(top, a.ends[2 * (row * a.pieces + i)]);
    low = fminf(low, a.ends[2 * (row * a.pieces + i) + 1]);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    top = fmaxf(top, __shfl_xor(top, d));
    low = fminf(low, __shfl_xor(low, d));
  }
  const float t = a.t ? a.t[row] : 1.0f;
  s.top = top;
  s.c = 92.332482616893656877 / (double)t;
  s.infinite = top == INFINITY;
  s.min_w = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;
  // 52 ln 2 = 36.04 times t below the maximum weights end; a little more than the range, so that the last of it is in the last step
  const float range = fminf(top - low, 36.05f * t) * 1.00001f;
  s.step = range > 1e-30f ? (float)SMP_STEPS / range : 0.f;
  return s;
}
// What cuts a row.  few: so small a k that all it keeps is listed and ranked, and no step's mass is needed
struct SampleCut {
  int k;
  float p;
  bool by_count, by_mass, few;
};
__device__ __forceinline__ SampleCut cut_of(const SampleArgs& a, int row) {
  SampleCut c;
  c.k = a.k ? a.k[row] : 0;
  c.p = a.p ? a.p[row] : 1.0f;
  c.by_count = c.k > 0 && c.k < a.V;
  c.by_mass = c.p < 1.0f;
  c.few = c.by_count && c.k <= SMP_RANKED / 2;
  return c;
}
__device__ __forceinline__ bool greedy(const SampleArgs& a, int row) { return a.t && !(a.t[row] > 0.f); }

// ---- 1: ends of every piece -------------------------------------------------------------------------------------------------
template <int XT>
__global__ __launch_bounds__(SMP_WG) void sample_ends_kernel(SampleArgs a) {
  __shared__ float s_top[SMP_WG / 64], s_low[SMP_WG / 64];
  __shared__ int s_at[SMP_WG / 64];
  const int piece = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const SampleSpan<XT> span(a, row);
  int v0, v1;
  share(span.vecs, a.pieces, piece, SMP_WG / 64, wave, v0, v1);
  float top = -INFINITY, low = INFINITY;
  int at = 0x7fffffff;
  if (v1 >= 0)
    span.walk(v0, v1, [&](int i, const float (&v)[SampleSpan<XT>::N], int n) {
#pragma unroll
      for (int e = 0; e < SampleSpan<XT>::N; e++) {
        if (e >= n) break;
        if (v[e] > top) top = v[e], at = i + e;
        if (v[e] > -INFINITY) low = fminf(low, v[e]);
      }
    });
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const float o = __shfl_xor(top, d);
    const int oa = __shfl_xor(at, d);
    if (o > top || (o == top && oa < at)) top = o, at = oa;
    low = fminf(low, __shfl_xor(low, d));
  }
  if (lane == 0) s_top[wave] = top, s_low[wave] = low, s_at[wave] = at;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < SMP_WG / 64; w++) {
      if (s_top[w] > top) top = s_top[w], at = s_at[w];  // (waves are in the order of the index)
      low = fminf(low, s_low[w]);
    }
    const int to = row * a.pieces + piece;
    a.ends[2 * to] = top;
    a.ends[2 * to + 1] = low;
    a.top[to] = at;
  }
}

// ---- 2: counts and masses of the steps --------------------------------------------------------------------------------------
template <int XT>
__global__ __launch_bounds__(SMP_WG) void sample_steps_kernel(SampleArgs a) {
  __shared__ uint32_t s_count[SMP_STEPS];
  __shared__ unsigned long long s_mass[SMP_STEPS];
  const int piece = blockIdx.x, row = blockIdx.y;
  if (greedy(a, row)) return;
  __shared__ double s_table[64];
  const SampleCut cut = cut_of(a, row);
  if (!cut.by_count && !cut.by_mass) return;  // nothing is cut off
  const SampleScale s = scale_of(a, row, s_table);
  if (s.top == -INFINITY) return;
  const bool by_mass = cut.by_mass && !cut.few;
  for (int i = threadIdx.x; i < SMP_STEPS; i += SMP_WG) s_count[i] = 0, s_mass[i] = 0;
  __syncthreads();
  const SampleSpan<XT> span(a, row);
  int v0, v1;
  share(span.vecs, a.pieces, piece, SMP_WG / 64, threadIdx.x >> 6, v0, v1);
  if (v1 >= 0)
    span.walk(v0, v1, [&](int, const float (&v)[SampleSpan<XT>::N], int n) {
#pragma unroll
      for (int e = 0; e < SampleSpan<XT>::N; e++) {
        const int step = e < n ? s.step_of(v[e]) : SMP_STEPS;
        if (step < SMP_STEPS) {
          atomicAdd(&s_count[step], 1u);
          if (by_mass) atomicAdd(&s_mass[step], (unsigned long long)(s.weight(v[e]) * a.unit + 0.5));
        }
      }
    });
  __syncthreads();
  const int64_t to = ((int64_t)row * a.pieces + piece) * SMP_STEPS;
  for (int i = threadIdx.x; i < SMP_STEPS; i += SMP_WG) {
    a.count[to + i] = s_count[i];
    a.mass[to + i] = s_mass[i];
  }
}

// inclusive sums over the workgroup, thread by thread
template <typename T, int WG>
__device__ __forceinline__ T running(T v, T* s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = v;
  __syncthreads();
  for (int w = 0; w < WG / 64; w++)
    if (w < wave) v += s_wave[w];
  return v;
}

// ---- 3: the border's steps, sums in front of them, a list of what is in them ---------------------------------------------------
template <int XT>
__global__ __launch_bounds__(SMP_WG) void sample_border_kernel(SampleArgs a) {
  static_assert(SMP_WG == SMP_STEPS, "a thread per step");
  __shared__ unsigned long long s_wave[SMP_WG / 64];
  __shared__ unsigned long long s_mass[SMP_STEPS];
  __shared__ uint32_t s_count[SMP_STEPS];
  __shared__ int s_first[2];
  __shared__ uint32_t s_list[SMP_WG / 64];
  __shared__ double s_sum[SMP_WG / 64];
  const int piece = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (greedy(a, row)) return;
  __shared__ double s_table[64];
  const SampleCut cut = cut_of(a, row);
  const int k = cut.k;
  const float p = cut.p;
  const bool by_count = cut.by_count, by_mass = cut.by_mass && !cut.few;
  // (all pieces' steps are on their way at once: one after the other they were 14 us)
  uint32_t counts_of[SMP_PIECES];
  unsigned long long mass_of[SMP_PIECES];
  if (by_count || by_mass) {
    const int64_t at = (int64_t)row * a.pieces * SMP_STEPS + tid;
#pragma unroll
    for (int i = 0; i < SMP_PIECES; i++) {
      const int64_t from = at + (int64_t)min(i, a.pieces - 1) * SMP_STEPS;
      counts_of[i] = a.count[from];
      mass_of[i] = by_mass ? a.mass[from] : 0;
    }
  }
  const SampleScale s = scale_of(a, row, s_table);
  if (s.top == -INFINITY) return;
  SampleRow r = {SMP_STEPS, SMP_STEPS, 0, 0, 0, 0, 0, 0};
  uint32_t mine = 0;  // elements of step tid in the pieces in front of this one
  if (by_count || by_mass) {
    unsigned long long count = 0, mass = 0;
#pragma unroll
    for (int i = 0; i < SMP_PIECES; i++) {
      if (i >= a.pieces) break;
      if (i < piece) mine += counts_of[i];
      count += counts_of[i];
      mass += mass_of[i];
    }
    const unsigned long long counts = running<unsigned long long, SMP_WG>(count, s_wave), masses = running<unsigned long long, SMP_WG>(mass, s_wave);
    s_count[tid] = (uint32_t)counts;
    s_mass[tid] = masses;
    if (tid < 2) s_first[tid] = SMP_STEPS;
    __syncthreads();
    auto up_to = [&](int step, bool m) -> unsigned long long { return step <= 0 ? 0 : m ? s_mass[step - 1] : s_count[step - 1]; };  // in front of a step
    if (by_count && counts >= (unsigned long long)k && counts - count < (unsigned long long)k) s_first[0] = tid;
    __syncthreads();
    r.cut = s_first[0] < SMP_STEPS;
    r.hi = s_first[0];
    r.mass = s_mass[SMP_STEPS - 1];
    if (cut.few) {
      r.lo = 0;
      r.hi = min(r.hi, SMP_STEPS - 1);
    } else if (by_mass) {  // with a cut by count the mass of what it keeps is only known to be that in front of step hi or more
      const double target = (double)p * (double)(r.cut ? up_to(r.hi, true) : r.mass);
      if ((double)masses >= target && (tid == 0 || (double)(masses - mass) < target)) atomicMin(&s_first[1], tid);
      __syncthreads();
      r.lo = min(s_first[1], r.cut ? r.hi : SMP_STEPS - 1);
      if (!r.cut) r.hi = r.lo;
    } else {
      r.lo = r.hi;
    }
    if (r.lo < SMP_STEPS) {
      r.above = (uint32_t)up_to(r.lo, false);
      r.mass_above = up_to(r.lo, true);
      r.listed = (uint32_t)(up_to(r.hi + 1, false) - r.above);
    } else {
      r.hi = SMP_STEPS - 1;
    }
    __syncthreads();
    mine = tid >= r.lo && tid <= r.hi ? mine : 0;
  }
  // where this piece's part of the list begins (and the weights' table is there)
  running<unsigned long long, SMP_WG>(mine, s_wave);
  uint32_t from = 0;
  for (int w = 0; w < SMP_WG / 64; w++) from += (uint32_t)s_wave[w];

  const SampleSpan<XT> span(a, row);
  constexpr int N = SampleSpan<XT>::N;
  int v0, v1;
  share(span.vecs, a.pieces, piece, SMP_WG / 64, wave, v0, v1);
  double sum = 0.0;
  uint32_t listed = 0;
  if (v1 >= 0)
    span.walk(v0, v1, [&](int, const float (&v)[N], int n) {
#pragma unroll
      for (int e = 0; e < N; e++) {
        const int step = e < n ? s.step_of(v[e]) : SMP_STEPS;
        if (step < r.lo) {
          const double w = s.weight(v[e]);
          sum += s.heavy(w) ? w : 0.0;
        } else if (step <= r.hi && step < SMP_STEPS) {
          listed++;
        }
      }
    });
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    sum += __shfl_xor(sum, d);
    listed += __shfl_xor(listed, d);
  }
  if (lane == 0) s_sum[wave] = sum, s_list[wave] = listed;
  __syncthreads();
  if (tid == 0) {
    double all = 0.0;
    for (int w = 0; w < SMP_WG / 64; w++) all += s_sum[w];
    a.sum[row * a.pieces + piece] = all;
    a.from[row * a.pieces + piece] = from;
    if (piece == 0) a.row[row] = r;
  }
  if (listed == 0) return;
  uint32_t to = from;
  for (int w = 0; w < wave; w++) to += s_list[w];
  uint32_t* list = a.list + (int64_t)row * a.V;
  span.walk(v0, v1, [&](int i, const float (&v)[N], int n) {
    uint32_t in = 0;
#pragma unroll
    for (int e = 0; e < N; e++) {
      const int step = e < n ? s.step_of(v[e]) : SMP_STEPS;
      in |= (uint32_t)(step >= r.lo && step <= r.hi && step < SMP_STEPS) << e;
    }
    if (!__ballot(in != 0)) return;
    const uint32_t have = __popc(in);
    uint32_t up = have;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(up, d);
      if (lane >= d) up += o;
    }
    uint32_t put = to + up - have;
#pragma unroll
    for (int e = 0; e < N; e++)
      if (in >> e & 1) list[put++] = (uint32_t)(i + e);
    to += __shfl(up, 63);
  });
}

// ---- 4: the border, the piece, the token --------------------------------------------------------------------------------------
struct SampleBorder {
  uint32_t key, equals;  // what is above `key` is kept, and the first `equals` of what has it
  unsigned long long mass;  // of all that
};
template <int XT>
__global__ __launch_bounds__(SMP_LAST) void sample_token_kernel(SampleArgs a) {
  constexpr int W = SMP_LAST / 64, N = SampleSpan<XT>::N;
  __shared__ uint32_t s_count[SMP_BINS];
  __shared__ unsigned long long s_mass[SMP_BINS];
  __shared__ unsigned long long s_wave[W];
  __shared__ double s_sum[W];
  __shared__ uint32_t s_key[2];
  __shared__ int s_at;
  __shared__ unsigned long long s_bin[3];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (greedy(a, row)) {
    if (wave) return;
    float top = -INFINITY;
    int at = 0x7fffffff;
    for (int i = lane; i < a.pieces; i += 64) {
      const float o = a.ends[2 * (row * a.pieces + i)];
      if (o > top) top = o, at = a.top[row * a.pieces + i];  // (pieces are in the order of the index)
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      const float o = __shfl_xor(top, d);
      const int oa = __shfl_xor(at, d);
      if (o > top || (o == top && oa < at)) top = o, at = oa;
    }
    if (lane == 0) a.token[row] = top == -INFINITY ? -1 : at;
    return;
  }
  __shared__ double s_table[64];
  const SampleScale s = scale_of(a, row, s_table);
  if (s.top == -INFINITY) {
    if (tid == 0) a.token[row] = -1;
    return;
  }
  const SampleRow r = a.row[row];
  const SampleSpan<XT> span(a, row);
  const uint32_t* list = a.list + (int64_t)row * a.V;
  const SampleCut cut = cut_of(a, row);
  const float p = cut.p;
  __syncthreads();

  // The border among the listed elements: the `want`-th of them (mass < 0), or the first at which their mass and base reach `target`.  Every
  // round counts the elements of a range of keys in 2048 bins from above and goes on with one bin.
  auto units = [&](float v) { return (unsigned long long)(s.weight(v) * a.unit + 0.5); };
  auto border = [&](bool by_mass, unsigned long long want, double target, unsigned long long base) {
    __syncthreads();
    if (tid == 0) s_key[0] = 0xffffffffu, s_key[1] = 0;
    __syncthreads();
    uint32_t low = 0xffffffffu, high = 0;
    for (uint32_t i = tid; i < r.listed; i += SMP_LAST) {
      const uint32_t key = key_of(span.at((int)list[i]));
      low = min(low, key), high = max(high, key);
    }
    atomicMin(&s_key[0], low);
    atomicMax(&s_key[1], high);
    __syncthreads();
    low = s_key[0], high = s_key[1];
    unsigned long long counted = 0, mass = base;
    for (;;) {
      const uint32_t width = high - low;
      const int bits = width ? 32 - __clz(width) : 0, shift = max(0, bits - 11);
      __syncthreads();
      for (int i = tid; i < SMP_BINS; i += SMP_LAST) s_count[i] = 0, s_mass[i] = 0;
      if (tid == 0) s_at = SMP_BINS;
      __syncthreads();
      for (uint32_t i = tid; i < r.listed; i += SMP_LAST) {
        const float v = span.at((int)list[i]);
        const uint32_t key = key_of(v);
        if (key < low || key > high) continue;
        const uint32_t bin = (high - key) >> shift;
        atomicAdd(&s_count[bin], 1u);
        atomicAdd(&s_mass[bin], units(v));
      }
      __syncthreads();
      const unsigned long long c0 = s_count[2 * tid], c1 = s_count[2 * tid + 1], m0 = s_mass[2 * tid], m1 = s_mass[2 * tid + 1];
      const unsigned long long c = running<unsigned long long, SMP_LAST>(c0 + c1, s_wave) - c0 - c1 + counted, m = running<unsigned long long, SMP_LAST>(m0 + m1, s_wave) - m0 - m1 + mass;
      const bool first = by_mass ? c0 && (double)(m + m0) >= target : c + c0 >= want, second = by_mass ? c1 && (double)(m + m0 + m1) >= target : c + c0 + c1 >= want;
      if (first || second) atomicMin(&s_at, first ? 2 * tid : 2 * tid + 1);
      __syncthreads();
      const bool found = s_at < SMP_BINS;
      if (!found && tid == 0) {  // (the mass falls short by what rounding to units took: everything)
        s_bin[0] = counted, s_bin[1] = mass;
      }
      if (found && s_at >> 1 == tid) {
        s_bin[0] = s_at & 1 ? c + c0 : c;
        s_bin[1] = s_at & 1 ? m + m0 : m;
        s_bin[2] = s_at & 1 ? c1 : c0;
      }
      __syncthreads();
      if (!found) return SampleBorder{low, 0xffffffffu, ~0ull};
      counted = s_bin[0], mass = s_bin[1];
      const uint32_t in = (uint32_t)s_bin[2];
      high -= (uint32_t)s_at << shift;
      low = max(low, high - min(high, (1u << shift) - 1));
      if (shift == 0) {
        const unsigned long long w = units(of_key(high));
        const double over = w ? ceil((target - (double)mass) / (double)w) : (double)in;
        const uint32_t equals = by_mass ? (uint32_t)fmin(fmax(over, 1.0), (double)in) : (uint32_t)min((unsigned long long)in, want - counted);
        return SampleBorder{high, equals, mass + w * equals};
      }
    }
  };
  uint32_t edge_key = 0;  // what is above it is kept, and what equals it up to index `last`
  int last = 0x7fffffff;
  if (r.lo < SMP_STEPS && r.listed <= SMP_RANKED) {
    // Few: everyone's rank and the mass in front of it, by comparing all with all; lanes of an element share the others.
    __shared__ unsigned long long s_of[SMP_RANKED];
    __shared__ uint32_t s_element[SMP_RANKED];
    int size = 16;
    while (size < (int)r.listed) size <<= 1;
    const int share_ = SMP_LAST / size, e = tid / share_, part = tid % share_;  // 2 .. 64 lanes
    if (tid < SMP_RANKED) {
      const float v = tid < (int)r.listed ? span.at((int)list[tid]) : -INFINITY;
      s_element[tid] = key_of(v);
      s_of[tid] = tid < (int)r.listed ? units(v) : 0;
    }
    if (tid < 2) s_key[tid] = 0;
    if (tid < 3) s_bin[tid] = 0;
    __syncthreads();
    const uint32_t key = s_element[e];
    const unsigned long long own = s_of[e];
    uint32_t rank = 0;
    unsigned long long before = 0;
    for (int i = part; i < (int)r.listed; i += share_) {
      const uint32_t o = s_element[i];
      const bool front = o > key || (o == key && i < e);
      rank += front;
      before += front ? s_of[i] : 0;
    }
    for (int d = 1; d < share_; d <<= 1) {
      rank += __shfl_xor(rank, d);
      before += __shfl_xor(before, d);
    }
    rank += r.above;
    before += r.mass_above;
    const bool here = e < (int)r.listed && part == 0;
    if (here && (r.cut ? rank == (uint32_t)cut.k - 1 : rank == r.above + r.listed - 1)) {  // the last that the count leaves: its number, the mass up to it
      s_key[0] = e;
      s_bin[0] = before + own;
    }
    __syncthreads();
    const double target = (double)p * (double)(r.cut || cut.few ? s_bin[0] : r.mass);
    if (cut.by_mass && here && (!r.cut || rank < (uint32_t)cut.k) && (double)before < target && (double)(before + own) >= target) {  // at most one
      s_key[0] = e;
      s_bin[1] = 1;
    }
    // (a mass of nothing or less is reached in front of the first, which is kept all the same)
    if (cut.by_mass && here && rank == 0 && !(target > 0.0)) s_key[0] = e;
    __syncthreads();
    edge_key = s_element[s_key[0]];
    last = (int)list[s_key[0]];
  } else if (r.lo < SMP_STEPS) {
    SampleBorder edge = {0, 0xffffffffu, 0};
    unsigned long long mass = r.mass;
    if (r.cut) {
      edge = border(false, (unsigned long long)a.k[row] - r.above, 0.0, r.mass_above);
      mass = edge.mass;
    }
    if (cut.by_mass) {
      const SampleBorder e = border(true, 0, (double)p * (double)mass, r.mass_above);
      if (!r.cut || e.key > edge.key || (e.key == edge.key && e.equals < edge.equals)) edge = e;
    }
    edge_key = edge.key;
    // the index of the last equal that is kept (the list is in the order of the index)
    if (edge.equals != 0xffffffffu) {
    __syncthreads();
    if (tid == 0) s_at = 0x7fffffff;
    const uint32_t per = (r.listed + SMP_LAST - 1) / SMP_LAST, i0 = min(r.listed, tid * per), i1 = min(r.listed, i0 + per);
    unsigned long long have = 0;
    for (uint32_t i = i0; i < i1; i++) have += key_of(span.at((int)list[i])) == edge.key;
    const unsigned long long up = running<unsigned long long, SMP_LAST>(have, s_wave);
    if (up >= edge.equals && up - have < edge.equals) {
      unsigned long long n = up - have;
      for (uint32_t i = i0; i < i1; i++)
        if (key_of(span.at((int)list[i])) == edge.key && ++n == edge.equals) s_at = (int)list[i];
    }
    __syncthreads();
    last = s_at;
    }
  }
  auto kept = [&](int i, float v) {  // the weight of a kept element, 0 of another
    const int step = s.step_of(v);
    if (step >= SMP_STEPS || step > r.hi) return 0.0;
    if (step >= r.lo) {
      const uint32_t key = key_of(v);
      if (key < edge_key || (key == edge_key && i > last)) return 0.0;
    }
    const double w = s.weight(v);
    return s.heavy(w) ? w : 0.0;
  };
  // sums of the pieces, and the one in which the running sum passes u of all
  double target = 0.0, before = 0.0;
  int piece = -1;
  {
    __shared__ double s_piece[64];
    for (int i = wave; i < a.pieces; i += W) {
      const uint32_t i0 = a.from[row * a.pieces + i], i1 = i + 1 < a.pieces ? a.from[row * a.pieces + i + 1] : r.listed;
      double sum = 0.0;
      if (r.lo < SMP_STEPS)
        for (uint32_t j = i0 + lane; j < i1; j += 64) sum += kept((int)list[j], span.at((int)list[j]));
#pragma unroll
      for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
      if (lane == 0) s_piece[i] = sum + a.sum[row * a.pieces + i];
    }
    __syncthreads();
    double total = 0.0, run = 0.0;
    for (int i = 0; i < a.pieces; i++) total += s_piece[i];
    target = (double)a.u[row] * total;
    for (int i = 0; i < a.pieces; i++) {
      const double next = run + s_piece[i];
      if (s_piece[i] > 0.0 && (piece < 0 || !(before + s_piece[piece] > target))) piece = i, before = run;
      run = next;
    }
  }
  if (piece < 0) {
    if (tid == 0) a.token[row] = -1;
    return;
  }
  // the same among the piece's waves, then among the elements of one
  int v0, v1;
  share(span.vecs, a.pieces, piece, W, wave, v0, v1);
  double sum = 0.0;
  if (v1 >= 0)
    span.walk(v0, v1, [&](int i, const float (&v)[N], int n) {
#pragma unroll
      for (int e = 0; e < N; e++)
        if (e < n) sum += kept(i + e, v[e]);
    });
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  int chosen = -1;
  double run = before, start = before;
  for (int w = 0; w < W; w++) {
    const double next = run + s_sum[w];
    if (s_sum[w] > 0.0 && (chosen < 0 || !(start + s_sum[chosen] > target))) chosen = w, start = run;
    run = next;
  }
  if (chosen < 0 && tid == 0) a.token[row] = -1;
  if (wave != chosen) return;
  int token = -1, at_last = -1;
  double passed = start;
  span.walk(v0, v1, [&](int i, const float (&v)[N], int n) {
    if (token >= 0) return;
    double w[N], mine = 0.0;
    int heaviest = -1;
#pragma unroll
    for (int e = 0; e < N; e++) {
      w[e] = e < n ? kept(i + e, v[e]) : 0.0;
      mine += w[e];
      if (w[e] > 0.0) heaviest = i + e;
    }
    const uint64_t any = __ballot(mine > 0.0);
    if (!any) return;
    double up = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double o = __shfl_up(up, d);
      if (lane >= d) up += o;
    }
    const uint64_t over = __ballot(mine > 0.0 && passed + up > target);
    at_last = __shfl(heaviest, 63 - __clzll(any));
    if (over) {
      const int who = __builtin_ctzll(over);
      double in = passed + up - mine;
      int mine_at = heaviest;  // (rounding: the lane's last)
#pragma unroll
      for (int e = N - 1; e >= 0; e--) {
        double to = in;
        for (int f = 0; f <= e; f++) to += w[f];
        if (w[e] > 0.0 && to > target) mine_at = i + e;
      }
      token = __shfl(mine_at, who);
    }
    passed += __shfl(up, 63);
  });
  if (lane == 0) a.token[row] = token >= 0 ? token : at_last;
}

// ---- host side ------------------------------------------------------------------------------------------------------------------
// Pieces of a row: enough workgroups for the chip, of 4096 logits at least, and SMP_PIECES at most (launch 3 adds up the steps of all pieces in every one)
static int sample_pieces(int64_t rows, int64_t V) {
  const int64_t most = (V + 4095) / 4096, want = (1024 + rows - 1) / rows;
  const int64_t n = want < most ? want : most;
  return (int)(n > SMP_PIECES ? SMP_PIECES : n);
}
static size_t sample_room(int64_t rows, int64_t V, int pieces) {
  const size_t rp = (size_t)rows * pieces;
  return align_up(rp * (SMP_STEPS * 12 + 8 + 4 + 8 + 4) + (size_t)rows * sizeof(SampleRow), 16) + (size_t)rows * V * 4;
}

}  // namespace mllmhip

using namespace mllmhip;

MLLM_API size_t mllm_hip_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > (1 << 24) || rows > 65535) return 0;
  return sample_room(rows, vocab, sample_pieces(rows, vocab));
}

MLLM_API int mllm_hip_sample(const void* logits, int dtype, int64_t row_stride, int64_t rows, int64_t vocab, const float* u, const float* temperature,
                             const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens, void* workspace, size_t workspace_bytes,
                             void* stream) {
  if ((dtype != MLLM_HIP_F32 && dtype != MLLM_HIP_BF16) || rows < 0 || vocab < 1 || row_stride < 0) return MLLM_HIP_E_BADARG;
  if (vocab > (1 << 24) || rows > 65535) return MLLM_HIP_E_SHAPE;
  if (rows == 0) return 0;
  if (!logits || !u || !tokens || !workspace) return MLLM_HIP_E_BADARG;
  auto al = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (!al(logits, dtype == MLLM_HIP_F32 ? 4 : 2) || !al(u, 4) || !al(temperature, 4) || !al(top_k, 4) || !al(top_p, 4) || !al(min_p, 4) || !al(tokens, 4) || !al(workspace, 16))
    return MLLM_HIP_E_ALIGN;
  const int pieces = sample_pieces(rows, vocab);
  if (workspace_bytes < sample_room(rows, vocab, pieces)) return MLLM_HIP_E_BADARG;
  SampleArgs a = {};
  a.x = logits;
  a.stride = row_stride;
  a.rows = (int)rows;
  a.V = (int)vocab;
  a.pieces = pieces;
  a.u = u;
  a.t = temperature;
  a.p = top_p;
  a.min_p = min_p;
  a.k = top_k;
  a.token = tokens;
  int bits = 0;
  while ((1ll << bits) < vocab) bits++;
  a.unit = (double)(1ull << (62 - bits));
  const size_t rp = (size_t)rows * pieces;
  char* w = reinterpret_cast<char*>(workspace);
  a.mass = reinterpret_cast<uint64_t*>(w);
  a.sum = reinterpret_cast<double*>(w + rp * SMP_STEPS * 8);
  a.row = reinterpret_cast<SampleRow*>(a.sum + rp);
  a.count = reinterpret_cast<uint32_t*>(a.row + rows);
  a.ends = reinterpret_cast<float*>(a.count + rp * SMP_STEPS);
  a.top = reinterpret_cast<int*>(a.ends + 2 * rp);
  a.from = reinterpret_cast<uint32_t*>(a.top + rp);
  a.list = reinterpret_cast<uint32_t*>(w + sample_room(rows, vocab, pieces) - (size_t)rows * vocab * 4);
  const dim3 grid((unsigned)pieces, (unsigned)rows);
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto ends, auto steps, auto border, auto token) {
    hipLaunchKernelGGL(ends, grid, dim3(SMP_WG), 0, st, a);
    if (top_k || top_p) hipLaunchKernelGGL(steps, grid, dim3(SMP_WG), 0, st, a);
    hipLaunchKernelGGL(border, grid, dim3(SMP_WG), 0, st, a);
    hipLaunchKernelGGL(token, dim3((unsigned)rows), dim3(SMP_LAST), 0, st, a);
  };
  if (dtype == MLLM_HIP_F32)
    go(sample_ends_kernel<MLLM_HIP_F32>, sample_steps_kernel<MLLM_HIP_F32>, sample_border_kernel<MLLM_HIP_F32>, sample_token_kernel<MLLM_HIP_F32>);
  else
    go(sample_ends_kernel<MLLM_HIP_BF16>, sample_steps_kernel<MLLM_HIP_BF16>, sample_border_kernel<MLLM_HIP_BF16>, sample_token_kernel<MLLM_HIP_BF16>);
  return (int)hipGetLastError();
}
