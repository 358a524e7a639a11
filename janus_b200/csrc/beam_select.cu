// The continuations that a step of beam search goes on with and the ones that end.
//
// Beam b of a request has score s_b and logits x_b over the vocabulary; a continuation (b, v) is worth
//   s_b + x_bv - log sum_u exp x_bu.
// The K best that are no stop token go on; a stop token among the K best of all ends its beam's text.  A beam's best continuation
// stays in the beam's row, so that cache rows and states move only where a beam is lost; the others take the rows left, in order.
//
// Three launches.  The first reads every logit once and does nothing but keep, in registers, each thread's largest one and its sum
// of exponentials.  In the second a block a beam finds the beam's K best: the K-th largest of the threads' maxima bounds the K-th
// largest logit of the row from below, and only the few threads' numbers at or above it are looked at again (from L2).  The third,
// a block a request, joins its beams.  64 requests of 8 beams over 128,256 tokens: 58 us, the first 44.  (With vectors of 16 bytes,
// of which the second fetches twice the memory, 60.  With the second step done by each block of the first launch 63 us: memory
// stood still meanwhile; with a warp a beam in the third 76.  With fewer launches, the last block of a row or of a request going on
// by a ticket: 61 by two, 65 by one, whose blocks that only read are fewer at a time; one request 12.8 and 13.6 us, by three 11.8.)
// Within a beam the order is that of the logits (equal ones: the lowest token first), which no rounding touches; between beams it is
// that of the totals.  The first launch makes each power, and adds up to 16 of them, in 32 bits: a power's exponent is within 2^6 and rounded
// twice, so that a logarithm is off by 2 * 2^-19 log(2) + 2^-21 < 3.3e-6 (in practice some 5e-8), and differently for equal rows that begin at
// different places of a vector.  Scores are given with that.  Where it could decide between two beams, the third launch sums their rows again in 64 bits.
#include <math_constants.h>
#include <stdio.h>
#include <stddef.h>
#include <string.h>

#include "common.cuh"

namespace {

typedef unsigned long long Key;      // a logit that sorts as a whole number, above the complement of its token: no two are equal; 0: none

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int WIDE_LOAD = 8;                              // numbers of a vector, 32 bytes
constexpr int VECTORS = 2;                                // that a thread has on its way at a time
constexpr int MOST_BEAMS = 32, MOST_STOPS = 32, MOST_RANGES = 8;
constexpr int AGAIN = 2;                                  // halves of vectors that a thread looks at again at a time
constexpr int ROOM = THREADS * 4 * AGAIN + MOST_BEAMS;            // candidates of a beam at a time
constexpr float FAR = 40.0f;                              // how far a power may lie above what a thread's sum is relative to
constexpr float WIDE = 1e8f;                              // powers beyond are made by 64-bit arithmetic
constexpr float NEAR = 256.0f;                            // powers of two as much below add nothing that 64 bits hold, however many there are

__device__ __forceinline__ unsigned sortable(float x) {   // of numbers, -0 taken as 0
  const unsigned u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float number(unsigned u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ Key key_of(float x, int token) { return ((Key)sortable(x) << 32) | (unsigned)~token; }
__device__ __forceinline__ float logit_of(Key k) { return number((unsigned)(k >> 32)); }
__device__ __forceinline__ int token_of(Key k) { return (int)~(unsigned)k; }

struct Stat {
  double sum;        // of exp(x) / 2^scale; of entries at +inf, if there are any
  double scale;
  double top;        // the largest number; -inf if there is none
};

struct Best {          // of a beam: score - log sum exp(x - top), and top, its largest logit; -inf, -inf: there is nothing
  double base, top;
};

struct Args {
  const float* logits;
  const float* scores;
  const int* stops;
  int* parents;
  int* tokens;
  float* next_scores;
  int* ended_parents;
  int* ended_tokens;
  float* ended_scores;
  float* maxima;      // [rows][ranges][THREADS]
  Stat* stats;        // [rows][ranges]
  Best* best;         // [rows]
  Key* keys;          // [rows][K]
  int R, K, V, S, ranges;
};

__device__ __forceinline__ bool dead(float score) { return !(score > -CUDART_INF_F); }

// exp(x) / 2^scale = 2^(x log2(e) - scale), two numbers at a time; log2(e) in two parts, the small one last, where the difference is small.
__device__ __forceinline__ jb::Pair powers(jb::Pair x, jb::Pair minus_scale) {
  constexpr float L = 1.44269504088896341f, L_LOW = 1.92596299112661746887e-8f;
  const jb::Pair p = jb::fma2(x, jb::pair(L_LOW, L_LOW), jb::fma2(x, jb::pair(L, L), minus_scale));
  float lo, hi;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(lo) : "f"(jb::lo(p)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(hi) : "f"(jb::hi(p)));
  return jb::pair(lo, hi);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
constexpr double LOG2E = 1.4426950408889634074;
// exp(x) as a power of two, rounded, so that the same numbers' powers are equal (a fused multiply-add would find their rounding)
__device__ __forceinline__ double power_of(double x) { return __dmul_rn(x, LOG2E); }
// A part's sum relative to exp(top), the largest number of all.
__device__ __forceinline__ double relative(const Stat& s, double top) {
  if (top == CUDART_INF) return s.top == top ? s.sum : 0.0;
  return s.top > -CUDART_INF ? s.sum * exp2(s.scale - power_of(top)) : 0.0;
}
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

struct Eight {
  float x[WIDE_LOAD];
};
__device__ __forceinline__ Eight load_eight(const float* at) {
  Eight v;
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v.x[0]), "=f"(v.x[1]), "=f"(v.x[2]), "=f"(v.x[3]), "=f"(v.x[4]), "=f"(v.x[5]), "=f"(v.x[6]), "=f"(v.x[7])
               : "l"(at));
  return v;
}

// A row of logits in vectors of 32 bytes; vector i holds numbers 8 i - lead .., of which the first and the last may lie outside the row.
// Range r of the row has vectors begin(r) .. begin(r + 1), its thread t those at begin(r) + t, + THREADS, ...
struct Row {
  const float* x;
  int lead, vectors, V, ranges;
  __device__ __forceinline__ Row(const Args& a, int row) : x(a.logits + (size_t)row * a.V), V(a.V), ranges(a.ranges) {
    lead = (int)(((uintptr_t)x >> 2) & (WIDE_LOAD - 1));
    vectors = (V + lead + WIDE_LOAD - 1) / WIDE_LOAD;
  }
  __device__ __forceinline__ int begin(int range) const { return (int)((long long)range * vectors / ranges); }
  __device__ __forceinline__ Eight load(int i) const {
    const int at = WIDE_LOAD * i - lead;
    if (at >= 0 && at + WIDE_LOAD <= V) return load_eight(x + at);
    Eight v;
#pragma unroll
    for (int e = 0; e < WIDE_LOAD; ++e) v.x[e] = at + e >= 0 && at + e < V ? x[at + e] : -CUDART_INF_F;
    return v;
  }
  __device__ __forceinline__ float4 load_half(int i) const {      // half i of the vectors
    const int at = 4 * i - lead;
    if (at >= 0 && at + 4 <= V) return *reinterpret_cast<const float4*>(x + at);
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = at + e >= 0 && at + e < V ? x[at + e] : -CUDART_INF_F;
    return make_float4(y[0], y[1], y[2], y[3]);
  }
};

__global__ void __launch_bounds__(THREADS) beam_rows_kernel(const Args a) {
  __shared__ double top_of[WARPS], sum_of[WARPS];
  jb::pdl_launch_dependents();
  const int row = blockIdx.x / a.ranges, range = blockIdx.x % a.ranges;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row x(a, row);
  const int first = x.begin(range), last = x.begin(range + 1);
  jb::pdl_wait();
  if (dead(a.scores[row])) return;                        // (the second launch asks for nothing of it)
  // ---- maximum and sum of the thread's numbers: vectors first + tid, + THREADS, ... ----
  // The sum is relative to a power of two near the first numbers' maximum, which is left where it is until one lies FAR above: what changes
  // with every new maximum would cost a warp as much as the numbers themselves.  Powers beyond WIDE below that are 0; where they are
  // all there is, where one lies just below -WIDE (beside larger ones it is worth something) or beyond WIDE, and where something is no
  // number, the thread goes over its numbers once more.
  float top = -CUDART_INF_F, scale = -CUDART_INF_F;
  bool wide = false;
  double sum = 0.0;
  auto take = [&](const Eight (&v)[VECTORS]) {
    float high = -CUDART_INF_F;                           // (what is no number is never the larger)
#pragma unroll
    for (int u = 0; u < VECTORS; ++u)
#pragma unroll
      for (int e = 0; e < WIDE_LOAD; e += 2) high = max3(high, v[u].x[e], v[u].x[e + 1]);
    top = fmaxf(top, high);
    const float power = high * (float)LOG2E;
    if (!(power >= -WIDE)) {
      wide |= power >= -WIDE - NEAR;
      return;
    }
    if (power > scale + FAR) {
      wide |= !(power <= WIDE);
      const float next = rintf(fminf(power, WIDE));
      sum *= exp2((double)scale - (double)next);          // (0 of nothing)
      scale = next;
    }
    jb::Pair s = jb::pair(0.0f, 0.0f), t = s;
    const jb::Pair minus = jb::pair(-scale, -scale), one = jb::pair(1.0f, 1.0f);
#pragma unroll
    for (int u = 0; u < VECTORS; ++u) {
#pragma unroll
      for (int e = 0; e < WIDE_LOAD; e += 4) {
        s = jb::fma2(powers(jb::pair(v[u].x[e], v[u].x[e + 1]), minus), one, s);
        t = jb::fma2(powers(jb::pair(v[u].x[e + 2], v[u].x[e + 3]), minus), one, t);
      }
    }
    sum += (double)((jb::lo(s) + jb::hi(s)) + (jb::lo(t) + jb::hi(t)));
  };
  const int whole0 = x.lead > 0 ? 1 : 0, whole1 = min(last, (x.V + x.lead) / WIDE_LOAD);     // vectors that lie inside the row
  for (int i0 = first + tid; i0 < last; i0 += THREADS * VECTORS) {
    Eight v[VECTORS];
    if (i0 >= whole0 && i0 + (VECTORS - 1) * THREADS < whole1) {
      const float* at = x.x - x.lead + (size_t)i0 * WIDE_LOAD;
#pragma unroll
      for (int u = 0; u < VECTORS; ++u) v[u] = load_eight(at + u * THREADS * WIDE_LOAD);
    } else {
#pragma unroll
      for (int u = 0; u < VECTORS; ++u) {
#pragma unroll
        for (int e = 0; e < WIDE_LOAD; ++e) v[u].x[e] = -CUDART_INF_F;
        if (i0 + u * THREADS < last) v[u] = x.load(i0 + u * THREADS);
      }
    }
    take(v);
  }
  Stat mine{sum, (double)scale, (double)top};
  if (wide || sum != sum || (scale == -CUDART_INF_F && top > -CUDART_INF_F)) {
    mine.sum = 0.0, mine.scale = power_of(mine.top);
    for (int i = first + tid; i < last; i += THREADS) {
      const Eight v = x.load(i);
      const float* y = v.x;
#pragma unroll
      for (int e = 0; e < WIDE_LOAD; ++e)
        if (y[e] > -CUDART_INF_F) mine.sum += top == CUDART_INF_F ? (y[e] == top ? 1.0 : 0.0) : exp((double)y[e] - mine.top);
    }
  }
  // ---- the range's sum, relative to its largest number ----
  const double warp_top = warp_max(mine.top);
  if (lane == 0) top_of[warp] = warp_top;
  __syncthreads();
  double all = top_of[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) all = fmax(all, top_of[w]);
  sum = relative(mine, all);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sum_of[warp] = sum;
  __syncthreads();
  const size_t list = (size_t)row * a.ranges + range;
  if (tid == 0) {
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += sum_of[w];
    a.stats[list] = Stat{s, power_of(all), all};
  }
  a.maxima[list * THREADS + tid] = top;
}

// A logit's distance from its row's largest; beside entries at +inf, 0 for those and -inf for others.
__device__ __forceinline__ double worth(float x, double top) {
  return top == CUDART_INF ? (x == CUDART_INF_F ? 0.0 : -CUDART_INF) : (double)x - top;
}

// The numbers of a warp, the largest in lane 0.
__device__ __forceinline__ float warp_sorted(float k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, k, o);
      const bool wants_more = ((lane & size) == 0) == ((lane & o) == 0);
      if ((other > k) == wants_more) k = other;
    }
  }
  return k;
}

__global__ void __launch_bounds__(THREADS) beam_best_kernel(const Args a) {
  __shared__ Key found[ROOM];          // the best so far, then what came
  __shared__ float heads[THREADS];
  __shared__ unsigned short chosen[MOST_RANGES * THREADS];    // threads of the first launch whose numbers are looked at again
  __shared__ float edge;
  __shared__ int n_found, n_chosen;
  __shared__ int stops[MOST_STOPS];
  jb::pdl_launch_dependents();
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.K;
  const Row x(a, row);
  if (tid < K) found[tid] = 0;
  if (tid == 0) edge = -CUDART_INF_F, n_found = K, n_chosen = 0;
  jb::pdl_wait();
  const float score = a.scores[row];
  if (dead(score)) {
    if (tid < K) a.keys[(size_t)row * K + tid] = 0;
    if (tid == 0) a.best[row] = Best{-CUDART_INF, -CUDART_INF};
    return;
  }
  if (tid < a.S) stops[tid] = a.stops[tid];
  float maxima[MOST_RANGES], top = -CUDART_INF_F;
#pragma unroll
  for (int r = 0; r < MOST_RANGES; ++r) {
    maxima[r] = r < a.ranges ? a.maxima[((size_t)row * a.ranges + r) * THREADS + tid] : -CUDART_INF_F;
    top = fmaxf(top, maxima[r]);
  }
  // ---- the bound: a stop token is at most one thread's maximum ----
  const int wanted = K + a.S, per_warp = min(wanted, 32);
  const float sorted = warp_sorted(top);
  if (lane < per_warp) heads[warp * per_warp + lane] = sorted;
  __syncthreads();
  if (tid < WARPS * per_warp && heads[tid] > -CUDART_INF_F) {
    const float mine = heads[tid];
    int above = 0, level = 0;                             // larger ones, equal ones
#pragma unroll 8
    for (int i = 0; i < WARPS * per_warp; ++i) above += heads[i] > mine, level += heads[i] == mine;
    if (above < wanted && above + level >= wanted) edge = mine;   // (all who are level write the same)
  }
  if (warp == WARPS - 1) {                                // ... and, by a warp with nothing to do, the row's sum
    Stat s{0.0, -CUDART_INF, -CUDART_INF};
    if (lane < a.ranges) s = a.stats[(size_t)row * a.ranges + lane];
    const double most = warp_max(s.top);
    double sum = relative(s, most);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) a.best[row] = most > -CUDART_INF ? Best{(double)score - log(sum), most} : Best{-CUDART_INF, -CUDART_INF};
  }
  __syncthreads();
  const float least = edge;                               // -inf: fewer threads than that have a number
#pragma unroll
  for (int r = 0; r < MOST_RANGES; ++r)
    if (maxima[r] >= least && maxima[r] > -CUDART_INF_F) chosen[atomicAdd(&n_chosen, 1)] = (unsigned short)(r * THREADS + tid);
  __syncthreads();
  // ---- their numbers at or above it, in rounds of two halves of vectors a thread (one or two, unless many maxima are equal) ----
  const int each = 2 * ((x.vectors + a.ranges - 1) / a.ranges / THREADS + 1), n = n_chosen * each;  // halves of a thread's vectors, at most
  Key bound = 0;                       // the K-th best so far, 0 while there are fewer
  for (int j0 = 0; j0 < n; j0 += THREADS * AGAIN) {
    float4 v[AGAIN];
    int half[AGAIN];                   // its number in the row; -1: none
#pragma unroll
    for (int u = 0; u < AGAIN; ++u) {
      const int j = j0 + u * THREADS + tid;
      half[u] = -1;
      if (j < n) {
        const int slot = chosen[j / each], range = slot / THREADS, i = x.begin(range) + slot % THREADS + j % each / 2 * THREADS;
        if (i < x.begin(range + 1)) half[u] = 2 * i + j % each % 2, v[u] = x.load_half(half[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < AGAIN; ++u) {
      if (half[u] >= 0) {
        const float y[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (y[e] >= least && y[e] > -CUDART_INF_F) {
            const int token = 4 * half[u] - x.lead + e;
            const Key k = key_of(y[e], token);
            bool stop = false;
            for (int s = 0; s < a.S; ++s) stop |= stops[s] == token;
            if (k > bound && !stop) found[atomicAdd(&n_found, 1)] = k;
          }
        }
      }
    }
    // (rounds whose numbers leave room for the next one's are put in order later)
    const bool last = j0 + THREADS * AGAIN >= n, full = __syncthreads_or(n_found > ROOM - 4 * AGAIN * THREADS) != 0;
    if (!full && !last) continue;
    // the K best of what was there and what came, in order: a key's place is the number of larger ones
    const int m = n_found;
    Key k[(ROOM + THREADS - 1) / THREADS];
    int place[(ROOM + THREADS - 1) / THREADS];
#pragma unroll
    for (int u = 0; u < (ROOM + THREADS - 1) / THREADS; ++u) {
      place[u] = K;
      if (u * THREADS >= m) continue;
      if (tid + u * THREADS < m) {
        k[u] = found[tid + u * THREADS];
        int above = 0;
        for (int q = 0; q < m; ++q) above += found[q] > k[u];
        if (k[u] > 0) place[u] = above;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < (ROOM + THREADS - 1) / THREADS; ++u)
      if (place[u] < K) found[place[u]] = k[u];
    if (tid == 0) n_found = K;
    __syncthreads();
    bound = found[K - 1];
  }
  if (tid < K) a.keys[(size_t)row * K + tid] = found[tid];     // (0 where the row has fewer)
}

constexpr int JOIN_THREADS = 256;
constexpr double DOUBT = 1e-5;                            // more than the totals of two beams may be off together

// What a block of the third launch has in shared memory, by beam and place (of a beam's continuations, in order; of the stop tokens): beam * 32 +
// place.  Behind it, of as many numbers as beams ask for: see Lists.
struct Join {
  double base[MOST_BEAMS], top[MOST_BEAMS];               // see Best
  double score[MOST_BEAMS];
  double kth[MOST_BEAMS], head[MOST_BEAMS];
  double scratch[JOIN_THREADS / 32];
  int n_list, n_stop;
  unsigned doubtful;                                      // beams
};
struct Lists {
  double* totals;         // then the short list's in order
  double* short_total;
  Key* keys;
  Key* stop_key;
  int* short_at;
  int* on_at;             // the short list in order
  int* stop_at;
  __device__ __forceinline__ Lists(uint8_t* memory, int K) {
    const int n = 32 * K;
    totals = reinterpret_cast<double*>(memory), short_total = totals + n, keys = reinterpret_cast<Key*>(short_total + n), stop_key = keys + n;
    short_at = reinterpret_cast<int*>(stop_key + n), on_at = short_at + n, stop_at = on_at + n;
  }
};
constexpr int JOIN_BYTES = 32 * (8 + 8 + 8 + 8 + 4 + 4 + 4);              // a beam
static_assert(MOST_BEAMS * JOIN_BYTES + sizeof(Join) <= 48 * 1024, "the third launch's memory");

// A continuation's total in its beam's list.
__device__ __forceinline__ void put_total(Join& m, const Lists& l, int K, int b, int place, Key key, double base, double top) {
  const double total = key > 0 ? base + worth(logit_of(key), top) : -CUDART_INF;
  l.totals[b * 32 + place] = total;
  if (place == 0) m.head[b] = total;
  if (place == K - 1) m.kth[b] = total;
}

// From a request's continuations to what goes on and ends.  FIRST: beams are marked whose totals lie too near to one another's.
// (Its code comes from memory, as the logits have passed through the L2 cache since: loops stay loops, and beams and places are told apart
// without a division.  With loops unrolled and divisions 64 requests of 8 beams over 128,256 tokens took 63 to 65 us.)
template <bool FIRST>
__device__ __forceinline__ void join_beams(const Args& a, Join& m, uint8_t* memory, float x0) {
  const int r = blockIdx.x, K = a.K, S = a.S, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, back = JOIN_THREADS - 1 - tid;
  constexpr double doubt = FIRST ? DOUBT : 0.0;
  const Lists l(memory, K);
  const double* on = l.totals;
  if (tid == 0) m.n_list = m.n_stop = 0, m.doubtful = 0u;
  if (tid < K) {
    a.ended_parents[r * K + tid] = a.ended_tokens[r * K + tid] = -1;
    a.ended_scores[r * K + tid] = -CUDART_INF_F;
  }
  __syncthreads();
  // ---- the K best of all beams: at least K lie at or above the largest K-th of a beam, and above the least of the beams' best ----
  double edge = -CUDART_INF, least = CUDART_INF;
#pragma unroll 1
  for (int b = 0; b < K; ++b) edge = fmax(edge, m.kth[b]), least = fmin(least, m.head[b]);
  edge = fmax(edge, least) - doubt;
#pragma unroll 1
  for (int i = tid; i < 32 * K; i += JOIN_THREADS) {
    const double t = l.totals[i];
    if (lane < K && t > -CUDART_INF && t >= edge) {
      const int at = atomicAdd(&m.n_list, 1);
      l.short_total[at] = t;
      l.short_at[at] = i;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < m.n_list; i += JOIN_THREADS) {
    const double t = l.short_total[i];
    const int at = l.short_at[i];
    int before = 0;
#pragma unroll 2
    for (int j = 0; j < m.n_list; ++j) {                    // (a beam's keys are in order)
      const double u = l.short_total[j];
      before += u > t || (u == t && l.short_at[j] < at);
    }
    l.totals[before] = t, l.on_at[before] = at;
  }
  if (tid < K && tid >= m.n_list) l.totals[tid] = -CUDART_INF, l.on_at[tid] = 0;
  __syncthreads();
  const double last = on[K - 1] - doubt;
  if (FIRST) {                                              // (by the last warps; of near ones in a row, every beam has a neighbour of another)
#pragma unroll 1
    for (int i = back; i + 1 < m.n_list; i += JOIN_THREADS) {
      const double u = on[i + 1];
      const int b = l.on_at[i] >> 5, c = l.on_at[i + 1] >> 5;
      if (on[i] - u <= doubt && u >= last && b != c) atomicOr(&m.doubtful, 1u << b | 1u << c);
    }
  }
  // ---- stop tokens that stand among the K best ----
#pragma unroll 1
  for (int b = warp; b < K; b += JOIN_THREADS / 32) {
    if (lane >= S || !(m.base[b] > -CUDART_INF)) continue;
    const int stop = a.stops[lane];
    bool twice = false;
#pragma unroll 1
    for (int s = 0; s < lane; ++s) twice |= a.stops[s] == stop;
    if (stop < 0 || stop >= a.V || twice) continue;
    const float x = FIRST && b == warp ? x0 : a.logits[((size_t)r * K + b) * a.V + stop];
    const double t = m.base[b] + worth(x, m.top[b]);
    if (!(x > -CUDART_INF_F) || !(t > -CUDART_INF) || t < last) continue;
    const int at = atomicAdd(&m.n_stop, 1);
    l.stop_key[at] = key_of(x, stop);
    l.stop_at[at] = b;
  }
  __syncthreads();
  auto stop_total = [&](int i) { return m.base[l.stop_at[i]] + worth(logit_of(l.stop_key[i]), m.top[l.stop_at[i]]); };
#pragma unroll 1
  for (int i = tid; i < m.n_stop; i += JOIN_THREADS) {
    const Key key = l.stop_key[i];
    const int b = l.stop_at[i];
    const double t = stop_total(i);
    int place = 0, before = 0;
#pragma unroll 1
    for (int j = -K; j < m.n_stop; ++j) {                   // continuations, then stop tokens
      const double u = j < 0 ? on[j + K] : stop_total(j);
      const int c = j < 0 ? l.on_at[j + K] >> 5 : l.stop_at[j];
      const Key other = j < 0 ? l.keys[l.on_at[j + K]] : l.stop_key[j];
      const bool front = u > t || (u == t && (c < b || (c == b && other > key)));
      before += front, place += front && j >= 0;
      if (FIRST && fabs(u - t) <= doubt && c != b) atomicOr(&m.doubtful, 1u << b | 1u << c);
    }
    if (before < K) {
      a.ended_parents[r * K + place] = b;
      a.ended_tokens[r * K + place] = token_of(key);
      a.ended_scores[r * K + place] = (float)t;
    }
  }
  // ---- rows: a beam's best continuation stays in the beam's row ----
  if (warp == 0) {
    const bool live = lane < K && on[lane] > -CUDART_INF;
    const int at = lane < K ? l.on_at[lane] : 0, parent = live ? at >> 5 : -1 - lane;
    const unsigned same = __match_any_sync(0xffffffffu, parent);
    const bool stays = live && (same & ((1u << lane) - 1u)) == 0;
    const unsigned kept = __reduce_or_sync(0xffffffffu, stays ? 1u << parent : 0u);
    const unsigned moves = __ballot_sync(0xffffffffu, lane < K && !stays);
    if (lane < K) {
      int row = parent;
      if (!stays) {
        unsigned left = ~kept;
#pragma unroll 1
        for (int n = __popc(moves & ((1u << lane) - 1u)); n > 0; --n) left &= left - 1;
        row = __ffs(left) - 1;
      }
      a.parents[r * K + row] = live ? parent : -1;
      a.tokens[r * K + row] = live ? token_of(l.keys[at]) : 0;
      a.next_scores[r * K + row] = (float)on[lane];
    }
  }
}

// The sum of exp(x - top) over a row, in 64 bits and in one order whatever the row's address.
__device__ __forceinline__ double row_sum(const float* x, int V, double top, double* scratch) {
  constexpr int AHEAD = 16;
  const int tid = threadIdx.x;
  double part[AHEAD] = {}, sum = 0.0;
#pragma unroll 1
  for (int i0 = 0; i0 < V; i0 += JOIN_THREADS * AHEAD) {
    float y[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) y[u] = i0 + u * JOIN_THREADS + tid < V ? x[i0 + u * JOIN_THREADS + tid] : -CUDART_INF_F;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const double d = worth(y[u], top);                  // (no number: nothing)
      part[u] += exp(y[u] > -CUDART_INF_F ? d : -CUDART_INF);
    }
  }
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) sum += part[u];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if ((tid & 31) == 0) scratch[tid >> 5] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < JOIN_THREADS / 32; ++w) sum += scratch[w];
  return sum;
}

// Where totals of two beams lie within DOUBT of one another and that may decide what goes on or ends, the first launch's sums do not tell them
// apart: those beams' rows are summed once more by the definition, and everything is ranked again.  (A call of its own, behind what has been
// written, so that nothing waits for it otherwise.)  Logits of the benchmark's distribution: no request of 768 with 8 beams over 128,256 tokens;
// where all 8 beams of 64 requests are equal 715 us for 58.
__device__ __noinline__ void join_again(const Args& a, Join& m, uint8_t* memory) {
  const int r = blockIdx.x, K = a.K, tid = threadIdx.x;
  for (unsigned left = m.doubtful; left != 0u; left &= left - 1) {
    const int b = __ffs(left) - 1;
    const double sum = row_sum(a.logits + ((size_t)r * K + b) * a.V, a.V, m.top[b], m.scratch);
    if (tid == 0) m.base[b] = m.score[b] - log(sum);
  }
  __syncthreads();
  const Lists l(memory, K);
  for (int b = tid >> 5, place = tid & 31; b < K; b += JOIN_THREADS / 32)
    if (place < K) put_total(m, l, K, b, place, l.keys[b * 32 + place], m.base[b], m.top[b]);
  join_beams<false>(a, m, memory, 0.0f);
}

// One block a request.
__global__ void __launch_bounds__(JOIN_THREADS) beam_join_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(16) uint8_t memory[];
  __shared__ Join m;
  const int r = blockIdx.x, K = a.K, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Lists l(memory, K);
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  if (tid < K) m.score[tid] = (double)a.scores[r * K + tid];          // (next_scores may be the same tensor)
#pragma unroll 1
  for (int b = warp; b < K; b += JOIN_THREADS / 32) {
    const Best best = a.best[r * K + b];
    if (lane == 0) m.base[b] = best.base, m.top[b] = best.top;
    if (lane < K) {
      const Key key = a.keys[((size_t)r * K + b) * K + lane];
      l.keys[b * 32 + lane] = key;
      put_total(m, l, K, b, lane, key, best.base, best.top);
    }
  }
  // (a stop token's logit is on its way meanwhile)
  const int stop = warp < K && lane < a.S ? a.stops[lane] : -1;
  const float x0 = stop >= 0 && stop < a.V ? a.logits[((size_t)r * K + warp) * a.V + stop] : -CUDART_INF_F;
  join_beams<true>(a, m, memory, x0);
  __syncthreads();
  if (m.doubtful != 0u) join_again(a, m, memory);
}

}  // namespace

// given: an Args in host memory.  Scratch: maxima R * K * ranges * 256 float32, stats R * K * ranges of 24 bytes,
// best R * K of 16, keys R * K * K of 8.
// Whether an output lies over an input or another output (next_scores may be scores itself).
static bool select_overlaps(const Args& a) {
  const char* at[9];
  static_assert(offsetof(Args, maxima) == sizeof(at), "nine tensors, the inputs first");
  memcpy(at, &a, sizeof(at));
  const size_t N = (size_t)a.R * a.K, n[9] = {N * a.V, N, (size_t)a.S, N, N, N, N, N, N};
  for (int i = 3; i < 9; ++i)
    for (int j = 0; j < i; ++j)
      if (n[j] > 0 && at[i] < at[j] + 4 * n[j] && at[j] < at[i] + 4 * n[i] && !(i == 5 && j == 1 && at[i] == at[j])) return true;
  return false;
}

JB_EXPORT int jb_beam_select(const void* given, cudaStream_t stream) {
  Args a;
  memcpy(&a, given, sizeof(a));
  const int R = a.R, K = a.K, V = a.V, S = a.S, ranges = a.ranges;
  JB_REFUSE(R < 1 || K < 1 || K > MOST_BEAMS || V < 1 || S < 0 || S > MOST_STOPS || ranges < 1 || ranges > MOST_RANGES ||
                (long long)R * K * ranges > 0x7fffffffLL || V > 0x7fffffff - 65536,
            "beam_select: %d requests of %d beams, vocabulary %d, %d stop tokens, %d ranges", R, K, V, S, ranges);
  if (select_overlaps(a)) return JB_ERR_OVERLAP;
  jb::Launch rows(dim3(R * K * ranges), dim3(THREADS), 0, stream);
  cudaError_t e = cudaLaunchKernelEx(&rows.c, beam_rows_kernel, a);
  if (e != cudaSuccess) return (int)e;
  jb::Launch best(dim3(R * K), dim3(THREADS), 0, stream);
  e = cudaLaunchKernelEx(&best.c, beam_best_kernel, a);
  if (e != cudaSuccess) return (int)e;
  const size_t memory = (size_t)K * JOIN_BYTES;
  jb::Launch join(dim3(R), dim3(JOIN_THREADS), memory, stream);
  return (int)cudaLaunchKernelEx(&join.c, beam_join_kernel, a);
}
