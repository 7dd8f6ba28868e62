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
// The row is read three times, from memory once (a row of 151 936 stays in the caches).  Weights and the sums of what is kept are fp64; the masses that
// find the border are added by atomics and therefore integers, in units of 2^-44 at 151 936 logits (2^-38 at 2^24): sums that do not depend on an order.  Each
// weight is rounded to a unit, so a mass is off by up to half a unit for every logit in it, 2^-28 of a row of 151 936 whose heaviest weighs 1; top_p itself has
// 24 bits.  Seen in the border: 75 000 equal logits of 2^-30 behind a peak, two of them more or fewer.
//
// What bounds it, per launch in us: one fp32 row of 151 936, k 50 and p .9: 5, 5, 9, 10 -- reads that wait for one another and barriers, nothing of the
// chip is busy.  128 bf16 rows, p .9: 13 (39 MB from memory), 31 (two atomics of LDS per logit and a weight of some 20 fp64 instructions), 28 (the
// read, weights in front of the border), 20 (one workgroup a row: rounds over the listed elements); with k 50 instead 13, 14, 18, 11.
#include "item8.h"

namespace mllmhip {

enum { SMP_STEPS = 512, SMP_WG = 512, SMP_BIN_BITS = 9, SMP_BINS = 1 << SMP_BIN_BITS, SMP_LAST = 1024, SMP_RANKED = 256, SMP_FEW = 256, SMP_HELD = 2048,
       SMP_PIECES = 16, SMP_HOLD = 5, SMP_FOUND = 128 };

struct SampleRow {  // what launch 3 finds out about a row
  int lo, mid, hi;  // the steps that may hold the border by mass are lo .. mid, the one by count is in is hi; lo = SMP_STEPS: everything is kept
  int cut;          // 1: the k-th is within the row's weights
  uint32_t listed;  // elements of steps lo .. mid and hi
  uint32_t want;    // which of the listed, in descending order, is the k-th
  uint64_t front;   // mass in front of step lo (in units)
  uint64_t front_k; // that and what lies between mid and hi: with the listed ones in front of the k-th, all that is in front of it
  uint64_t mass;    // of the row
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
  double* sum;      // [rows][pieces][waves]
  uint32_t* from;   // the same: where a wave's elements begin in the list
  uint32_t* list;   // [rows][V]
  SampleRow* row;
};

// a logit as the operator takes it: no number counts as -inf, -0 as 0
__device__ __forceinline__ float logit(float v) { return v != v ? -INFINITY : v + 0.0f; }
__device__ __forceinline__ uint32_t key_of(float v) {  // larger logits, larger keys
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// A row as 16-byte vectors of N logits: vector 0 ends where the first aligned one begins (it may be empty), the last one is what is left.
// Elements of a vector that the row does not have count as -inf.
template <int XT>
struct SampleSpan {
  static constexpr int N = XT == MLLM_HIP_F32 ? 4 : 8;
  const char* x;
  int V, lead, vecs;  // lead: elements that vector 0 lacks in front
  __device__ __forceinline__ SampleSpan(const SampleArgs& a, int row) {
    constexpr int wide = 16 / N;
    x = reinterpret_cast<const char*>(a.x) + row * a.stride * wide;
    V = a.V;
    lead = (int)(reinterpret_cast<uintptr_t>(x) & 15) / wide;
    vecs = (lead + V + N - 1) / N;
  }
  __device__ __forceinline__ float at(int i) const {
    return logit(XT == MLLM_HIP_F32 ? reinterpret_cast<const float*>(x)[i] : bf16_to_f32(reinterpret_cast<const uint16_t*>(x)[i]));
  }
  __device__ __forceinline__ int first_of(int vec) const { return vec * N - lead; }
  __device__ __forceinline__ bool whole(int vec) const { return first_of(vec) >= 0 && first_of(vec) + N <= V; }
  __device__ __forceinline__ u32x4 load(int vec) const { return *reinterpret_cast<const u32x4*>(x + (int64_t)first_of(vec) * (16 / N)); }
  __device__ __forceinline__ u32x4 part(int vec) const {  // element by element
    const int i = first_of(vec);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < N; e++) {
      const bool in = i + e >= 0 && i + e < V;
      if (XT == MLLM_HIP_F32) w[e % 4] = in ? reinterpret_cast<const uint32_t*>(x)[i + e] : 0xff800000u;
      else w[e / 2 % 4] |= (uint32_t)(in ? reinterpret_cast<const uint16_t*>(x)[i + e] : 0xff80u) << (e % 2 * 16);
    }
    return u32x4{w[0], w[1], w[2], w[3]};
  }
  // as they are in memory: whoever takes them compares them so that no number is like -inf, and -0 like 0
  static __device__ __forceinline__ void logits(const u32x4& r, float (&v)[N]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (XT == MLLM_HIP_F32) {
        v[e] = __uint_as_float(w[e]);
      } else {
        v[2 * e % N] = __uint_as_float(w[e] << 16);
        v[(2 * e + 1) % N] = __uint_as_float(w[e] & 0xffff0000u);
      }
    }
  }
};
// A wave's vectors of a row, in the order of the index.  They go through LDS (H vectors a lane at a time, on their way all at once while those before
// them are worked on), so that the loop over them is short: code is fetched anew by every launch, and unrolled over registers these kernels ran for as long
// as that took.
template <int XT, int H>
struct SampleWalk {
  typedef SampleSpan<XT> Span;
  static constexpr int N = Span::N;
  const Span& span;
  u32x4* lds;  // [H][64] of this wave
  int v0, v1, held, asked;
  u32x4 r[H];  // on their way
  __device__ __forceinline__ SampleWalk(const Span& span_, u32x4* lds_, int pieces, int p, int waves, int wave) : span(span_), lds(lds_ + wave * H * 64), held(-1), asked(-1) {
    const int per = (span.vecs + pieces - 1) / pieces, a = min(span.vecs, p * per), b = min(span.vecs, a + per), each = (b - a + waves - 1) / waves;
    v0 = min(b, a + wave * each);
    v1 = min(b, v0 + each);
  }
  __device__ __forceinline__ void ask(int from) {
    asked = from;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < H; j++) {
      const int vec = min(from + j * 64 + lane, v1 - 1);
      r[j] = span.whole(vec) ? span.load(vec) : u32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void hold(int from) {
    if (held == from) return;
    if (asked != from) ask(from);
    held = from;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < H; j++) lds[j * 64 + lane] = r[j];
#pragma unroll 1
    for (int end = 0; end < 2; end++) {  // the row's first and last vector
      const int vec = end ? span.vecs - 1 : 0;
      if (vec >= from && vec < min(v1, from + H * 64) && !span.whole(vec) && (vec - from) % 64 == lane) lds[vec - from] = span.part(vec);
    }
  }
  // f(i, v): a lane's elements i .. i + N - 1; every lane comes along, with -inf where it has none
  template <typename F>
  __device__ __forceinline__ void operator()(F&& f) {
    const int lane = threadIdx.x & 63;
    for (int b = v0; b < v1; b += H * 64) {
      hold(b);
      if (b + H * 64 < v1) ask(b + H * 64);
#pragma unroll 1
      for (int at = b + lane, j = 0; j < H && b + j * 64 < v1; j++, at += 64) {
        float v[N];
        Span::logits(lds[j * 64 + lane], v);
        if (at >= v1) {
#pragma unroll
          for (int e = 0; e < N; e++) v[e] = -INFINITY;
        }
        f(span.first_of(at), v);
      }
    }
  }
};

// 2^(j / 64), rounded to nearest
__device__ const double g_pow64[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0};
typedef __attribute__((address_space(3))) double* lds_double;
// A row's weights: its maximum, what divides its logits, and the steps
struct SampleScale {
  float top, step;
  double c;       // 64 / (t ln 2)
  double at;      // the maximum; 2^1000 where it is infinite, and infinite logits count as that: its equals weigh 1, the rest nothing
  float min_w;
  lds_double table;  // 2^(j / 64), j = 0 .. 63
  // exp((v - top) / t) = 2^(n / 64) e^(r ln 2 / 64) with n + r = (v - top) c, |r| <= 1/2: the table, a power of two and five terms of the series (the
  // sixth is under 2^-54).  Off by 2^-52 and what rounding (v - top) c leaves of up to 36, 2^-47; the library's exp of a quotient took three times as long.
  // No branches: eight of them are worked on at a time.
  __device__ __forceinline__ double weight(float v) const {
    const double y = fmax((fmin((double)v, 0x1p1000) - at) * c, -3400.0);
    const double n = rint(y), r = (y - n) * 0.010830424696249145;
    const int i = (int)n;
    double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    e = fma(r, e, 1.0 / 6.0);
    e = fma(r, e, 0.5);
    e = fma(r, e, 1.0);
    e = fma(r, e, 1.0);
    e = __builtin_ldexp(e * table[i & 63], i >> 6);
    return y > -3328.0 ? e : 0.0;  // 52 * 64: below 2^-52
  }
  // the step of a logit; SMP_STEPS: its weight is below 2^-52 (inf - inf is step 0)
  __device__ __forceinline__ int step_of(float v) const { return (int)fminf(fmaxf((top - v) * step, 0.0f), (float)SMP_STEPS); }
  // a weight in whole units, 2^51 to the weight of 1 at most: added to 2^52 they are the low bits of the sum
  __device__ __forceinline__ unsigned long long units(float v, double unit) const {
    return (unsigned long long)__double_as_longlong(fma(weight(v), unit, 0x1p52)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ bool heavy(double w) const { return w > 0.0 && w >= (double)min_w; }
};
// What every launch reads of a row first, all of it asked for at once: settings, and a piece's ends per lane
struct SampleIn {
  float t, p, min_p, top, low;
  int k;
  __device__ __forceinline__ SampleIn(const SampleArgs& a, int row) {
    const int lane = threadIdx.x & (SMP_PIECES - 1);  // every SMP_PIECES lanes have all pieces
    const f32x2 ends = reinterpret_cast<const f32x2*>(a.ends)[row * a.pieces + min(lane, a.pieces - 1)];
    t = a.t ? a.t[row] : 1.0f;
    k = a.k ? a.k[row] : 0;
    p = a.p ? a.p[row] : 1.0f;
    min_p = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;
    top = ends.x;
    low = ends.y;
  }
  __device__ __forceinline__ bool greedy() const { return !(t > 0.f); }
};
// (the caller waits for the other waves before it takes a weight)
__device__ __forceinline__ SampleScale scale_of(const SampleIn& in, lds_double table) {
  SampleScale s;
  if (threadIdx.x < 64) table[threadIdx.x] = g_pow64[threadIdx.x];
  s.table = table;
  float top = in.top, low = in.low;
#pragma unroll
  for (int d = SMP_PIECES / 2; d; d >>= 1) {
    top = fmaxf(top, __shfl_xor(top, d));
    low = fminf(low, __shfl_xor(low, d));
  }
  s.top = top + 0.0f;
  s.c = 92.332482616893656877 / (double)in.t;
  s.at = top == INFINITY ? 0x1p1000 : (double)top;
  s.min_w = in.min_p;
  // 52 ln 2 = 36.04 times t below the maximum weights end; a little more than the range, so that the last of it is in the last step
  const float range = fminf(fminf(top - low, 36.05f * in.t) * 1.00001f, 3e38f);
  s.step = range > 1e-30f && top < INFINITY ? (float)SMP_STEPS / range : 1.0f;
  return s;
}
// What cuts a row.  few: so small a k that all it keeps is listed and ranked, and no step's mass is needed
struct SampleCut {
  int k;
  float p;
  bool by_count, by_mass, few;
  __device__ __forceinline__ SampleCut(const SampleArgs& a, const SampleIn& in) {
    k = in.k;
    p = in.p;
    by_count = k > 0 && k < a.V;
    by_mass = p < 1.0f;
    few = by_count && k <= SMP_FEW;
  }
};

// ---- 1: ends of every piece -------------------------------------------------------------------------------------------------
template <int XT>
__global__ __launch_bounds__(SMP_WG) void sample_ends_kernel(SampleArgs a) {
  __shared__ __align__(16) u32x4 s_x[SMP_WG * SMP_HOLD];
  __shared__ float s_top[SMP_WG / 64], s_low[SMP_WG / 64];
  __shared__ int s_at[SMP_WG / 64];
  const int piece = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const SampleSpan<XT> span(a, row);
  SampleWalk<XT, SMP_HOLD> walk(span, s_x, a.pieces, piece, SMP_WG / 64, wave);
  float top = -INFINITY, low = INFINITY;
  int at = 0x7fffffff;
  walk([&](int i, const float (&v)[SampleSpan<XT>::N]) {
#pragma unroll
    for (int e = 0; e < SampleSpan<XT>::N; e++) {
      if (v[e] > top) top = v[e], at = i + e;
      low = fminf(low, v[e] > -INFINITY ? v[e] : INFINITY);
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
#pragma unroll 1
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
__global__ __launch_bounds__(SMP_LAST) void sample_steps_kernel(SampleArgs a) {
  __shared__ __align__(16) u32x4 s_x[SMP_LAST * 3];
  __shared__ uint32_t s_count[SMP_STEPS];
  __shared__ unsigned long long s_mass[SMP_STEPS];
  const int piece = blockIdx.x, row = blockIdx.y;
  __shared__ double s_table[64];
  const SampleSpan<XT> span(a, row);
  SampleWalk<XT, 3> walk(span, s_x, a.pieces, piece, SMP_LAST / 64, threadIdx.x >> 6);
  const SampleIn in(a, row);
  const SampleCut cut(a, in);
  if (walk.v0 < walk.v1) walk.hold(walk.v0);
  if (in.greedy() || (!cut.by_count && !cut.by_mass)) return;  // nothing is cut off
  const SampleScale s = scale_of(in, (lds_double)s_table);
  if (s.top == -INFINITY) return;
  const bool by_mass = cut.by_mass && !cut.few;
  for (int i = threadIdx.x; i < SMP_STEPS; i += SMP_LAST) s_count[i] = 0, s_mass[i] = 0;
  __syncthreads();
  walk([&](int, const float (&v)[SampleSpan<XT>::N]) {
    constexpr int N = SampleSpan<XT>::N;
    const float v0 = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v[0])));
    bool same = true;
#pragma unroll
    for (int e = 0; e < N; e++) same &= v[e] == v0;
    if (!~__ballot(same)) {  // (64 N atomics on one address took 1.2 ms of a call of 128 rows of 151936 equal logits)
      const int step = s.step_of(v0);
      if (step < SMP_STEPS && (threadIdx.x & 63) == 0) {
        atomicAdd(&s_count[step], 64u * N);
        if (by_mass) atomicAdd(&s_mass[step], s.units(v0, a.unit) * (64 * N));
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < N; e++) {
      const int step = s.step_of(fmaxf(v[e], -INFINITY));  // (no number: -inf)
      if (step < SMP_STEPS) {
        atomicAdd(&s_count[step], 1u);
        if (by_mass) atomicAdd(&s_mass[step], s.units(v[e], a.unit));
      }
    }
  });
  __syncthreads();
  const int64_t to = ((int64_t)row * a.pieces + piece) * SMP_STEPS;
  for (int i = threadIdx.x; i < SMP_STEPS; i += SMP_LAST) {
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

// inclusive sums of counts and masses over the workgroup, thread by thread
template <int WG>
__device__ __forceinline__ void running2(uint32_t& c, unsigned long long& m, uint32_t* s_c, unsigned long long* s_m) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t oc = __shfl_up(c, d);
    const unsigned long long om = __shfl_up(m, d);
    if (lane >= d) c += oc, m += om;
  }
  if (lane == 63) s_c[wave] = c, s_m[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WG / 64; w++)
    if (w < wave) c += s_c[w], m += s_m[w];
}

__device__ __forceinline__ bool in_list(const SampleRow& r, int step) { return (step >= r.lo && step <= r.mid) || (r.lo < SMP_STEPS && step == r.hi); }

// The steps as logits: an element's step is below S where its logit is at least the least one that has such a step, found by search over the keys (a
// logit's step never grows with the logit), 16 lanes for each of the four.  One or two comparisons take the place of the step of every element: a call
// of 128 rows of 151936 bf16 logits, k 50, took 82 us with the steps and 73 with these.
struct SampleBounds {
  float front, mid, before, last;  // of the elements in front of the list (those of steps below lo), up to mid, in front of hi, up to hi
  __device__ __forceinline__ SampleBounds(const SampleScale& s, const SampleRow& r) {
    const int lane = threadIdx.x & 63, j = lane & 15;
    const bool cut = r.lo < SMP_STEPS;
    const int below = lane < 16 || !cut ? r.lo : lane < 32 ? r.mid + 1 : lane < 48 ? r.hi : r.hi + 1;
    uint32_t no = key_of(-INFINITY), yes = key_of(s.top);  // the keys that have no such step, and that have one (of step 0 and more)
    // (about where it is, which saves most of the rounds)
    const float away = (float)below / s.step, about = s.top - away, slack = (fabsf(s.top) + fabsf(away)) * 0x1p-21f;
    if (s.step_of(about - slack) >= below) no = key_of(about - slack);
    if (about + slack < s.top && s.step_of(about + slack) < below) yes = key_of(about + slack);
    while (__ballot(yes - no > 1)) {
      const uint64_t width = yes - no;
      const uint32_t probe = no + (uint32_t)(width * (j + 1) >> 4);
      const uint32_t found = (uint32_t)(__ballot(j == 15 || s.step_of(of_key(probe)) < below) >> (lane & 48)) & 0xffff;
      const int at = __builtin_ctz(found);
      yes = no + (uint32_t)(width * (at + 1) >> 4);
      no = no + (uint32_t)(width * at >> 4);
    }
    const float least = below > 0 ? of_key(yes) : NAN;  // (nothing compares as that or more)
    auto of = [&](int l) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(least), l)); };
    front = of(0), mid = of(16), before = of(32), last = of(48);
  }
  // of the elements from hi's on that are not in front, the listed ones
  __device__ __forceinline__ uint64_t listed(float v, uint64_t some) const { return some & ~(__ballot(v >= before) & ~__ballot(v >= mid)); }
};

// ---- 3: the border's steps, sums in front of them, a list of what is in them ---------------------------------------------------
template <int XT>
__global__ __launch_bounds__(SMP_WG) void sample_border_kernel(SampleArgs a) {
  static_assert(SMP_WG == SMP_STEPS, "a thread per step");
  constexpr int N = SampleSpan<XT>::N;
  __shared__ __align__(16) u32x4 s_x[SMP_WG * SMP_HOLD];
  __shared__ unsigned long long s_wave[SMP_WG / 64];
  __shared__ unsigned long long s_mass[SMP_STEPS];
  __shared__ uint32_t s_count[SMP_STEPS];
  __shared__ int s_first[2], s_last;
  __shared__ uint32_t s_list[SMP_WG / 64];
  __shared__ uint32_t s_found[SMP_WG / 64][SMP_FOUND];  // the first of a wave's listed elements: mostly all
  __shared__ float s_dense[SMP_WG * (1 + N)];
  const int piece = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ double s_table[64];
  const SampleSpan<XT> span(a, row);
  SampleWalk<XT, SMP_HOLD> walk(span, s_x, a.pieces, piece, SMP_WG / 64, wave);
  const SampleIn given(a, row);
  const SampleCut cut(a, given);
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
  if (walk.v0 < walk.v1) walk.hold(walk.v0);
  if (given.greedy()) return;
  const SampleScale s = scale_of(given, (lds_double)s_table);
  if (s.top == -INFINITY) return;
  SampleRow r = {SMP_STEPS, SMP_STEPS - 1, SMP_STEPS - 1, 0, 0, 0, 0, 0, 0};
  uint32_t mine = 0;  // elements of step tid in the pieces in front of this one
  if (by_count || by_mass) {
    uint32_t count = 0;
    unsigned long long mass = 0;
#pragma unroll
    for (int i = 0; i < SMP_PIECES; i++) {
      if (i >= a.pieces) break;
      if (i < piece) mine += counts_of[i];
      count += counts_of[i];
      mass += mass_of[i];
    }
    uint32_t counts = count;
    unsigned long long masses = mass;
    running2<SMP_WG>(counts, masses, s_list, s_wave);
    s_count[tid] = counts;
    s_mass[tid] = masses;
    if (tid < 2) s_first[tid] = SMP_STEPS;
    if (tid == 2) s_last = SMP_STEPS - 1;
    __syncthreads();
    auto up_to = [&](int step, bool m) -> unsigned long long { return step <= 0 ? 0 : m ? s_mass[step - 1] : s_count[step - 1]; };  // in front of a step
    if (by_count && counts >= (uint32_t)k && counts - count < (uint32_t)k) s_first[0] = tid;
    __syncthreads();
    r.cut = s_first[0] < SMP_STEPS;
    r.mass = s_mass[SMP_STEPS - 1];
    if (r.cut) r.hi = r.mid = s_first[0];
    if (cut.few) {
      r.lo = 0;
    } else if (by_mass) {  // with a cut by count the mass of what it keeps is only known to be between that in front of step hi and with it
      const double least = (double)p * (double)(r.cut ? up_to(r.hi, true) : r.mass), most = (double)p * (double)(r.cut ? up_to(r.hi + 1, true) : r.mass);
      if ((double)masses >= least && (tid == 0 || (double)(masses - mass) < least)) atomicMin(&s_first[1], tid);
      if ((double)masses >= most && (tid == 0 || (double)(masses - mass) < most)) atomicMin(&s_last, tid);
      __syncthreads();
      r.mid = min(s_last, r.hi);
      r.lo = min(s_first[1], r.mid);
      if (!r.cut) r.hi = r.mid;
    } else if (r.cut) {
      r.lo = r.hi;
    }
    if (r.lo < SMP_STEPS) {
      const int before = min(r.mid + 1, r.hi);  // the listed steps in front of hi are lo .. before - 1
      const uint32_t front_listed = (uint32_t)(up_to(before, false) - up_to(r.lo, false));
      r.front = up_to(r.lo, true);
      r.listed = front_listed + (uint32_t)(up_to(r.hi + 1, false) - up_to(r.hi, false));
      if (r.cut) {
        r.want = (uint32_t)k - (uint32_t)up_to(r.hi, false) + front_listed;
        r.front_k = up_to(r.hi, true) - (up_to(before, true) - r.front);
      } else {
        r.want = r.listed;  // (a small k that does not cut: fewer than k have a weight, and all of them are listed)
        r.front_k = r.front;
      }
    }
    __syncthreads();
    mine = in_list(r, tid) ? mine : 0;
  }
  // where this piece's part of the list begins (and the weights' table is there)
#pragma unroll
  for (int d = 32; d; d >>= 1) mine += __shfl_xor(mine, d);
  __syncthreads();
  if (lane == 0) s_list[wave] = mine;
  __syncthreads();
  uint32_t from = 0;
#pragma unroll
  for (int w = 0; w < SMP_WG / 64; w++) from += s_list[w];
  __syncthreads();

  // Where few elements are in front of the border a weight of each lane would be one of them at a time: they are collected, 64 and more, first.
  float* dense = s_dense + wave * (64 + 64 * N);
  double sum = 0.0;
  uint32_t listed = 0, *found = s_found[wave];
  int waiting = 0;
  auto add = [&](int n) {
    const double w = s.weight(dense[waiting + lane]);
    sum += lane < n && s.heavy(w) ? w : 0.0;
  };
  const SampleBounds bound(s, r);
  walk([&](int i, const float (&v)[N]) {
    uint64_t front[N], some[N], any = 0, all = ~0ull, list = 0;
#pragma unroll
    for (int e = 0; e < N; e++) {
      front[e] = __ballot(v[e] >= bound.front);
      some[e] = __ballot(v[e] >= bound.last) & ~front[e];
      any |= front[e], all &= front[e], list |= some[e];
    }
    if (list) {
      uint32_t put = listed;  // (a lane's elements follow one another)
#pragma unroll
      for (int e = 0; e < N; e++) {
        some[e] = bound.listed(v[e], some[e]);
        put = __builtin_amdgcn_mbcnt_hi((uint32_t)(some[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some[e], put));
        listed += (uint32_t)__popcll(some[e]);
      }
#pragma unroll
      for (int e = 0; e < N; e++) {
        const bool in = some[e] >> lane & 1;
        if (in && put < SMP_FOUND) found[put] = (uint32_t)(i + e);
        put += in;
      }
    }
    if (!~all) {
#pragma unroll
      for (int e = 0; e < N; e++) {
        const double w = s.weight(v[e]);
        sum += s.heavy(w) ? w : 0.0;
      }
    } else if (any) {
#pragma unroll
      for (int e = 0; e < N; e++) {
        if (v[e] >= bound.front) dense[__builtin_amdgcn_mbcnt_hi((uint32_t)(front[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)front[e], waiting))] = v[e];
        waiting += __popcll(front[e]);
      }
      while (waiting >= 64) {
        waiting -= 64;
        add(64);
      }
    }
  });
  const int rest = waiting;
  waiting = 0;
  add(rest);
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) s_list[wave] = listed;
  __syncthreads();
  for (int w = 0; w < wave; w++) from += s_list[w];
  if (lane == 0) {
    const int to = (row * a.pieces + piece) * (SMP_WG / 64) + wave;
    a.sum[to] = sum;
    a.from[to] = from;
  }
  if (tid == 0 && piece == 0) a.row[row] = r;
  if (listed == 0) return;
  uint32_t to = from;
  uint32_t* list = a.list + (int64_t)row * a.V;
  if (listed <= SMP_FOUND) {
    for (uint32_t j = lane; j < listed; j += 64) list[to + j] = found[j];
    return;
  }
  walk([&](int i, const float (&v)[N]) {
    uint64_t in[N], any = 0;
#pragma unroll
    for (int e = 0; e < N; e++) any |= in[e] = __ballot(v[e] >= bound.last) & ~__ballot(v[e] >= bound.front);
    if (!any) return;
#pragma unroll
    for (int e = 0; e < N; e++) in[e] = bound.listed(v[e], in[e]);
    uint32_t put = to;  // (a lane's elements follow one another)
#pragma unroll
    for (int e = 0; e < N; e++) {
      put = __builtin_amdgcn_mbcnt_hi((uint32_t)(in[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in[e], put));
      to += (uint32_t)__popcll(in[e]);
    }
#pragma unroll
    for (int e = 0; e < N; e++)
      if (in[e] >> lane & 1) list[put++] = (uint32_t)(i + e);
  });
}

// ---- 4: the border, the piece, the token --------------------------------------------------------------------------------------
struct SampleBorder {
  uint32_t key;  // what is above is kept, and what equals it up to index `last`
  int last;
  unsigned long long mass;  // of all that
};
template <int XT>
__global__ __launch_bounds__(SMP_LAST) void sample_token_kernel(SampleArgs a) {
  constexpr int W = SMP_LAST / 64, N = SampleSpan<XT>::N;
  __shared__ uint32_t s_count[SMP_BINS];
  __shared__ unsigned long long s_mass[SMP_BINS];
  __shared__ unsigned long long s_wave[W];
  __shared__ double s_sum[W];
  __shared__ __align__(16) u32x4 s_x[SMP_LAST * 3];
  __shared__ uint32_t s_element[SMP_HELD], s_index[SMP_HELD];  // the list: keys, indexes and masses
  __shared__ unsigned long long s_of[SMP_HELD];
  struct __align__(16) Ranked {
    unsigned long long order, mass;  // the key, then the place in the list (the earlier the larger)
  };
  __shared__ Ranked s_rank[SMP_RANKED];
  __shared__ uint32_t s_ends[2];
  __shared__ int s_at;
  __shared__ unsigned long long s_bin[3];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const SampleIn in(a, row);
  const SampleRow r = a.row[row];  // (launch 3 writes none for a row it has nothing to do for)
  const float u_of = a.u[row];
  constexpr int WAVES = SMP_WG / 64;  // of launch 3
  const int part_of = row * a.pieces * WAVES + min(tid, a.pieces * WAVES - 1);
  const double own_sum = a.sum[part_of];
  const uint32_t own_from = a.from[part_of];
  if (in.greedy()) {
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
  const SampleScale s = scale_of(in, (lds_double)s_table);
  if (s.top == -INFINITY) {
    if (tid == 0) a.token[row] = -1;
    return;
  }
  const SampleSpan<XT> span(a, row);
  const uint32_t* list = a.list + (int64_t)row * a.V;
  const SampleCut cut(a, in);
  const float p = cut.p;
  __syncthreads();

  // The border among the listed elements: the `want`-th of them, or the first at which their mass and base reach `target`.  While more than SMP_RANKED are
  // left, every round counts a range of keys in SMP_BINS bins from above and goes on with one of them; the rest are ranked against one another.
  auto units = [&](float v) { return s.units(v, a.unit); };
  const bool kept_in_lds = r.listed <= SMP_HELD;
  if (r.lo < SMP_STEPS && kept_in_lds) {
    for (uint32_t i = tid; i < r.listed; i += SMP_LAST) {
      const uint32_t index = list[i];
      const float v = span.at((int)index);
      s_index[i] = index;
      s_element[i] = key_of(v);
      s_of[i] = units(v);
    }
  }
  auto element = [&](uint32_t i) { return kept_in_lds ? s_element[i] : key_of(span.at((int)list[i])); };
  auto mass_of = [&](uint32_t i, uint32_t key) { return kept_in_lds ? s_of[i] : units(of_key(key)); };
  auto index_of = [&](uint32_t i) {
    if (!kept_in_lds) return (int)list[i];
    int index = (int)s_index[i];
    asm volatile("" : "+v"(index));  // (merged with the other load it would be one from a generic address)
    return index;
  };
  bool all_ranked = false;  // the whole list, by the border by count: the one by mass finds the ranks where they are
  Ranked own = {0, 0};
  uint32_t rank = 0;
  unsigned long long in_front = 0;
  auto border = [&](bool by_mass, unsigned long long want, double target, unsigned long long base) __attribute__((always_inline)) {
    uint32_t low = 0, high = 0xffffffffu, left = r.listed;
    unsigned long long counted = 0, mass = base;
    bool narrowed = false;
    for (;;) {
      if (left <= SMP_RANKED) {
        // ranks and masses in front, by comparing all with all; lanes of an element share the others
        __syncthreads();
        const int n = (int)left;
        int size = 16;
        while (size < n) size <<= 1;
        const int share_ = SMP_LAST / size, e = tid / share_;  // 2 .. 64 lanes
        const bool live = e < n;
        if (tid < 2) s_bin[tid] = ~0ull;
        if (!all_ranked) {
          if (tid == 0) s_at = 0;
          __syncthreads();
          for (uint32_t i = tid; i < r.listed; i += SMP_LAST) {
            const uint32_t key = element(i);
            if (key < low || key > high) continue;
            s_rank[atomicAdd(&s_at, 1)] = Ranked{(unsigned long long)key << 32 | (0xffffffffu - i), mass_of(i, key)};
          }
          __syncthreads();
          own = s_rank[live ? e : 0];
          rank = 0;
          in_front = 0;
#pragma unroll 4
          for (int i = tid % share_; i < n; i += share_) {
            const Ranked o = s_rank[i];
            const bool front = o.order > own.order;
            rank += front;
            in_front += front ? o.mass : 0;
          }
          for (int d = 1; d < share_; d <<= 1) {
            rank += __shfl_xor(rank, d);
            in_front += __shfl_xor(in_front, d);
          }
          all_ranked = left == r.listed;
        } else {
          __syncthreads();
        }
        const unsigned long long before = in_front + mass;
        if (live && tid % share_ == 0) {
          // (a mass of nothing or less is reached in front of the first, which is kept all the same)
          const bool it = by_mass ? (double)(before + own.mass) >= target && ((double)before < target || (rank == 0 && counted == 0)) : counted + rank + 1 == want;
          if (it || rank + 1 == left) {
            atomicMin(&s_bin[0], (unsigned long long)(it ? 0 : 1) << 32 | (0xffffffffu - (uint32_t)own.order));  // the last where rounding to units leaves it short of the target
            if (it) s_bin[1] = before + own.mass;
          }
        }
        __syncthreads();
        const uint32_t i = (uint32_t)s_bin[0];
        return SampleBorder{element(i), index_of(i), s_bin[1]};
      }
      if (!narrowed) {  // the ends of the keys
        narrowed = true;
        __syncthreads();
        if (tid == 0) s_ends[0] = 0xffffffffu, s_ends[1] = 0;
        __syncthreads();
        uint32_t least = 0xffffffffu, most = 0;
        if (kept_in_lds) {
          for (uint32_t i = tid; i < r.listed; i += SMP_LAST) least = min(least, s_element[i]), most = max(most, s_element[i]);
        } else {
          for (uint32_t i = tid; i < r.listed; i += SMP_LAST * 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = span.at((int)list[min(i + j * SMP_LAST, r.listed - 1)]);
#pragma unroll
            for (int j = 0; j < 8; j++) least = min(least, key_of(v[j])), most = max(most, key_of(v[j]));
          }
        }
#pragma unroll 1
        for (int d = 32; d; d >>= 1) least = min(least, (uint32_t)__shfl_xor((int)least, d)), most = max(most, (uint32_t)__shfl_xor((int)most, d));
        if (lane == 0) {
          atomicMin(&s_ends[0], least);
          atomicMax(&s_ends[1], most);
        }
        __syncthreads();
        low = s_ends[0], high = s_ends[1];
      }
      if (low == high) {  // very many equal logits: the first so many of them, found by their number in the list, which is in the order of the index
        const unsigned long long w = units(of_key(high));
        const double over = w ? ceil((target - (double)mass) / (double)w) : (double)left;
        const unsigned long long equals = by_mass ? (unsigned long long)fmin(fmax(over, 1.0), (double)left) : want - counted;
        if (left == r.listed) return SampleBorder{high, index_of((uint32_t)equals - 1), mass + w * equals};
        __syncthreads();
        const uint32_t per = (r.listed + SMP_LAST - 1) / SMP_LAST, i0 = min(r.listed, tid * per), i1 = min(r.listed, i0 + per);
        unsigned long long have = 0;
        for (uint32_t i = i0; i < i1; i++) have += element(i) == high;
        const unsigned long long up = running<unsigned long long, SMP_LAST>(have, s_wave);
        if (up >= equals && up - have < equals) {
          unsigned long long n = up - have;
          for (uint32_t i = i0; i < i1; i++)
            if (element(i) == high && ++n == equals) s_at = index_of(i);
        }
        __syncthreads();
        return SampleBorder{high, s_at, mass + w * equals};
      }
      const uint32_t width = high - low;
      const int bits = width ? 32 - __clz(width) : 0, shift = max(0, bits - SMP_BIN_BITS);
      __syncthreads();
      for (int i = tid; i < SMP_BINS; i += SMP_LAST) s_count[i] = 0, s_mass[i] = 0;
      if (tid == 0) s_at = SMP_BINS;
      __syncthreads();
      for (uint32_t i = tid; i < r.listed; i += SMP_LAST) {
        const uint32_t key = element(i);
        if (key < low || key > high) continue;
        const uint32_t bin = (high - key) >> shift;
        const unsigned long long w = mass_of(i, key);
        const uint64_t here = __ballot(true);
        if (__ballot(key == (uint32_t)__builtin_amdgcn_readfirstlane(key)) == here) {  // (one address)
          if (lane == __builtin_ctzll(here)) {
            atomicAdd(&s_count[bin], (uint32_t)__popcll(here));
            atomicAdd(&s_mass[bin], w * __popcll(here));
          }
          continue;
        }
        atomicAdd(&s_count[bin], 1u);
        atomicAdd(&s_mass[bin], w);
      }
      __syncthreads();
      if (wave == 0) {  // a lane's bins, the lanes' sums, the lane that crosses, its bin
        constexpr int PER = SMP_BINS / 64;
        unsigned long long c = 0, m = 0;
#pragma unroll 1
        for (int j = 0; j < PER; j++) c += s_count[lane * PER + j], m += s_mass[lane * PER + j];
        const unsigned long long own_c = c, own_m = m;
#pragma unroll 1
        for (int d = 1; d < 64; d <<= 1) {
          const unsigned long long oc = __shfl_up(c, d), om = __shfl_up(m, d);
          if (lane >= d) c += oc, m += om;
        }
        c += counted, m += mass;
        const uint64_t over = __ballot(by_mass ? own_c && (double)m >= target : c >= want);
        if (over && lane == __builtin_ctzll(over)) {
          c -= own_c, m -= own_m;
#pragma unroll 1
          for (int j = lane * PER; j < (lane + 1) * PER; j++) {
            const unsigned long long bc = s_count[j], bm = s_mass[j];
            if (by_mass ? bc && (double)(m + bm) >= target : c + bc >= want) {
              s_at = j;
              s_bin[0] = c, s_bin[1] = m, s_bin[2] = bc;
              break;
            }
            c += bc, m += bm;
          }
        }
      }
      __syncthreads();
      const int found = s_at;
      if (found == SMP_BINS) return SampleBorder{low, 0x7fffffff, ~0ull};  // (the mass falls short by what rounding to units took: everything)
      counted = s_bin[0], mass = s_bin[1];
      left = (uint32_t)s_bin[2];
      high -= (uint32_t)found << shift;
      low = max(low, high - min(high, (1u << shift) - 1));
    }
  };
  uint32_t edge_key = 0;  // what is above it is kept, and what equals it up to index `last`
  int last = 0x7fffffff;
  if (r.lo < SMP_STEPS) {
    // by count first, which says what the mass is that top-p takes its part of; without a k that cuts: all, and its mass is known
    unsigned long long mass = r.mass;
    SampleBorder edge = {0, 0x7fffffff, 0};
#pragma unroll 1
    for (int by_mass = r.cut || cut.few ? 0 : 1; by_mass <= (cut.by_mass ? 1 : 0); by_mass++) {
      const SampleBorder e = border(by_mass, r.want, (double)p * (double)mass, by_mass ? r.front : r.front_k);
      if (e.key > edge.key || (e.key == edge.key && e.last < edge.last)) edge = e;
      mass = e.mass;
    }
    edge_key = edge.key;
    last = edge.last;
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
  if (r.lo == 0 && r.listed <= SMP_LAST) {  // all that is kept is in the list: an element per thread
    const double w = tid < (int)r.listed ? kept((int)s_index[tid], of_key(s_element[tid])) : 0.0;
    const double up = running<double, SMP_LAST>(w, s_sum);
    if (tid == 0) s_at = 0x7fffffff, s_ends[0] = 0;
    double total = 0.0;
    for (int i = 0; i < W; i++) total += s_sum[i];
    __syncthreads();
    if (w > 0.0) {
      atomicMax(&s_ends[0], (uint32_t)tid);
      if (up > (double)u_of * total) atomicMin(&s_at, tid);
    }
    __syncthreads();
    if (tid == 0) a.token[row] = (int)s_index[s_at < SMP_LAST ? s_at : s_ends[0]];
    return;
  }
  // sums of the parts that launch 3 had a wave for, and the part in which the running sum passes u of all
  __shared__ double s_part[SMP_PIECES * WAVES];
  __shared__ uint32_t s_from[SMP_PIECES * WAVES + 1];
  __shared__ double s_start[2];
  const int parts = a.pieces * WAVES;
  if (r.lo == SMP_STEPS) {
    if (tid < parts) s_part[tid] = own_sum;
  } else if (kept_in_lds) {  // every listed weight by a thread of its own, then every part by one
    for (uint32_t i = tid; i < r.listed; i += SMP_LAST) s_of[i] = (unsigned long long)__double_as_longlong(kept((int)s_index[i], of_key(s_element[i])));
    if (tid < parts) s_from[tid] = own_from;
    if (tid == 0) s_from[parts] = r.listed;
    __syncthreads();
    if (tid < parts) {
      double sum = own_sum;
      for (uint32_t i = s_from[tid], end = s_from[tid + 1]; i < end; i++) sum += __longlong_as_double((long long)s_of[i]);
      s_part[tid] = sum;
    }
  } else {
    if (tid < parts) s_from[tid] = own_from, s_part[tid] = own_sum;
    if (tid == 0) s_from[parts] = r.listed;
    __syncthreads();
    for (int i = wave; i < parts; i += W) {
      double sum = 0.0;
      for (uint32_t j = s_from[i] + lane; j < s_from[i + 1]; j += 64 * 4) {
        int index[4];
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) index[e] = (int)list[min(j + e * 64, r.listed - 1)];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = span.at(index[e]);
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (j + e * 64 < s_from[i + 1]) sum += kept(index[e], v[e]);
      }
#pragma unroll 1
      for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
      if (lane == 0) s_part[i] += sum;
    }
  }
  __syncthreads();
  // lane by lane two parts each: the first lane, then its part, whose end is beyond the target; the last of all with anything where rounding says none
  auto pick = [&](const double* part, int n, double target, double start) __attribute__((always_inline)) {
    const double x0 = 2 * lane < n ? part[2 * lane] : 0.0, x1 = 2 * lane + 1 < n ? part[2 * lane + 1] : 0.0;
    double up = x0 + x1;
#pragma unroll 1
    for (int d = 1; d < 64; d <<= 1) {
      const double o = __shfl_up(up, d);
      if (lane >= d) up += o;
    }
    if (target < 0.0) target = -target * __shfl(up, 63);  // (a part of all: below)
    const double front = start + up - x0 - x1;
    const bool first = x0 > 0.0 && front + x0 > target, second = x1 > 0.0 && start + up > target;
    const uint64_t over = __ballot(first || second), any = __ballot(x0 > 0.0 || x1 > 0.0);
    if (!any) return -1;
    const int who = over ? __builtin_ctzll(over) : 63 - __clzll(any);
    const bool one = over ? !first : x1 > 0.0;
    if (lane == who) s_start[0] = one ? front + x0 : front, s_start[1] = target;
    return 2 * who + (int)__shfl((int)one, who);
  };
  const double u = fmax((double)u_of, 1e-300);  // (0 asks for the first part with anything, as any number this small does)
  if (wave == 0) {
    const int at = pick(s_part, parts, -u, 0.0);
    if (lane == 0) s_at = at;
  }
  __syncthreads();
  const int part = s_at;
  if (part < 0) {
    if (tid == 0) a.token[row] = -1;
    return;
  }
  const double before = s_start[0], target = s_start[1];
  // the same among the runs of the part that this kernel's waves have, then among the elements of one
  SampleWalk<XT, 3> walk(span, s_x, a.pieces, part / WAVES, WAVES, part % WAVES);
  {
    const int each = (walk.v1 - walk.v0 + W * 64 - 1) / (W * 64) * 64, end = walk.v1;
    walk.lds = s_x + wave * 3 * 64;
    walk.v0 = min(end, walk.v0 + wave * each);
    walk.v1 = min(end, walk.v0 + each);
  }
  double sum = 0.0;
  walk([&](int i, const float (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; e++) sum += kept(i + e, logit(v[e]));
  });
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  const int chosen = pick(s_sum, W, target, before);  // (every wave: it writes the same)
  if (chosen < 0 && tid == 0) a.token[row] = -1;
  if (wave != chosen) return;
  const double start = s_start[0];
  int token = -1, at_last = -1;
  double passed = start;
  walk([&](int i, const float (&v)[N]) {
    if (token >= 0) return;
    double w[N], mine = 0.0;
    int heaviest = -1;
#pragma unroll
    for (int e = 0; e < N; e++) {
      w[e] = kept(i + e, logit(v[e]));
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
// Pieces of a row: two workgroups a CU, which is what launch 3's registers leave room for, of 4096 logits at least, and SMP_PIECES at most (launch 3 adds
// up the steps of all pieces in every one).  128 rows of 151936 bf16 logits, k 50 / p .9, with 384, 512 and 1024 workgroups: 76 / 122, 67 / 104, 75 / 109 us.
static int sample_pieces(int64_t rows, int64_t V) {
  const int64_t most = (V + 4095) / 4096, want = (512 + rows - 1) / rows;
  const int64_t n = want < most ? want : most;
  return (int)(n > SMP_PIECES ? SMP_PIECES : n);
}
static size_t sample_room(int64_t rows, int64_t V, int pieces) {
  const size_t rp = (size_t)rows * pieces;
  return align_up(rp * (SMP_STEPS * 12 + 12 + 12 * (SMP_WG / 64)) + (size_t)rows * sizeof(SampleRow), 16) + (size_t)rows * V * 4;
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
  a.unit = (double)(1ull << (62 - bits < 51 ? 62 - bits : 51));
  const size_t rp = (size_t)rows * pieces;
  char* w = reinterpret_cast<char*>(workspace);
  a.mass = reinterpret_cast<uint64_t*>(w);
  a.sum = reinterpret_cast<double*>(w + rp * SMP_STEPS * 8);
  a.row = reinterpret_cast<SampleRow*>(a.sum + rp * (SMP_WG / 64));
  a.count = reinterpret_cast<uint32_t*>(a.row + rows);
  a.ends = reinterpret_cast<float*>(a.count + rp * SMP_STEPS);
  a.top = reinterpret_cast<int*>(a.ends + 2 * rp);
  a.from = reinterpret_cast<uint32_t*>(a.top + rp);
  a.list = reinterpret_cast<uint32_t*>(w + sample_room(rows, vocab, pieces) - (size_t)rows * vocab * 4);
  const dim3 grid((unsigned)pieces, (unsigned)rows);
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto ends, auto steps, auto border, auto token) {
    hipLaunchKernelGGL(ends, grid, dim3(SMP_WG), 0, st, a);
    if (top_k || top_p) hipLaunchKernelGGL(steps, grid, dim3(SMP_LAST), 0, st, a);
    hipLaunchKernelGGL(border, grid, dim3(SMP_WG), 0, st, a);
    hipLaunchKernelGGL(token, dim3((unsigned)rows), dim3(SMP_LAST), 0, st, a);
  };
  if (dtype == MLLM_HIP_F32)
    go(sample_ends_kernel<MLLM_HIP_F32>, sample_steps_kernel<MLLM_HIP_F32>, sample_border_kernel<MLLM_HIP_F32>, sample_token_kernel<MLLM_HIP_F32>);
  else
    go(sample_ends_kernel<MLLM_HIP_BF16>, sample_steps_kernel<MLLM_HIP_BF16>, sample_border_kernel<MLLM_HIP_BF16>, sample_token_kernel<MLLM_HIP_BF16>);
  return (int)hipGetLastError();
}
