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
// that of the totals, whose sum of exponentials is taken to 64 bits where threads meet: 32 bits would turn two beams round now and
// then.
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

// One block a request.  Dynamic memory: K * K continuations (total, key), their shortened list, and a list of K * S stop tokens.
__global__ void __launch_bounds__(JOIN_THREADS) beam_join_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t memory[];
  __shared__ double base[MOST_BEAMS], top_of[MOST_BEAMS];  // see Best
  __shared__ double kth[MOST_BEAMS], head[MOST_BEAMS];
  __shared__ double on[MOST_BEAMS];
  __shared__ int on_at[MOST_BEAMS];                        // beam * K + place
  __shared__ int n_list, n_stop;
  const int r = blockIdx.x, K = a.K, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, KK = K * K;
  double* totals = reinterpret_cast<double*>(memory);                    // [K][K]
  double* short_total = totals + KK;
  Key* keys = reinterpret_cast<Key*>(short_total + KK);                  // [K][K]
  Key* stop_key = keys + KK;                                             // [K * S]
  int* short_at = reinterpret_cast<int*>(stop_key + K * a.S);            // beam * K + place
  int* stop_at = short_at + KK;                                          // beam
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  if (tid < K) {
    const Best best = a.best[r * K + tid];
    base[tid] = best.base, top_of[tid] = best.top;
  }
  for (int i = tid; i < KK; i += JOIN_THREADS) keys[i] = a.keys[(size_t)r * KK + i];
  // (a stop token's logit is on its way meanwhile)
  const int b0 = a.S > 0 ? tid / a.S : K, stop0 = b0 < K ? a.stops[tid % a.S] : -1;
  const float x0 = b0 < K && stop0 >= 0 && stop0 < a.V ? a.logits[((size_t)r * K + b0) * a.V + stop0] : -CUDART_INF_F;
  auto total_of = [&](Key k, int b) { return base[b] + worth(logit_of(k), top_of[b]); };
  if (tid == 0) n_list = n_stop = 0;
  if (tid < K) {
    a.ended_parents[r * K + tid] = a.ended_tokens[r * K + tid] = -1;
    a.ended_scores[r * K + tid] = -CUDART_INF_F;
    on[tid] = -CUDART_INF;
    on_at[tid] = 0;
  }
  __syncthreads();
  for (int i = tid; i < KK; i += JOIN_THREADS) {
    const double total = keys[i] > 0 ? total_of(keys[i], i / K) : -CUDART_INF;
    totals[i] = total;
    if (i % K == 0) head[i / K] = total;
    if (i % K == K - 1) kth[i / K] = total;
  }
  __syncthreads();
  // ---- the K best of all beams: at least K lie at or above the largest K-th of a beam, and above the least of the beams' best ----
  double edge = -CUDART_INF, least = CUDART_INF;
  for (int b = 0; b < K; ++b) edge = fmax(edge, kth[b]), least = fmin(least, head[b]);
  edge = fmax(edge, least);
  for (int i = tid; i < KK; i += JOIN_THREADS) {
    if (totals[i] > -CUDART_INF && totals[i] >= edge) {
      const int at = atomicAdd(&n_list, 1);
      short_total[at] = totals[i];
      short_at[at] = i;
    }
  }
  __syncthreads();
  for (int i = tid; i < n_list; i += JOIN_THREADS) {
    const double t = short_total[i];
    const int at = short_at[i];
    int before = 0;
    for (int j = 0; j < n_list; ++j) {                    // (a beam's keys are in order)
      const double u = short_total[j];
      before += u > t || (u == t && short_at[j] < at);
    }
    if (before < K) on[before] = t, on_at[before] = at;
  }
  __syncthreads();
  // ---- stop tokens that stand among the K best ----
  for (int i = tid; i < K * a.S; i += JOIN_THREADS) {
    const int b = i / a.S, stop = a.stops[i % a.S];
    bool twice = false;
    for (int s = 0; s < i % a.S; ++s) twice |= a.stops[s] == stop;
    if (stop < 0 || stop >= a.V || twice || !(base[b] > -CUDART_INF)) continue;
    const float x = i == tid ? x0 : a.logits[((size_t)r * K + b) * a.V + stop];
    if (!(x > -CUDART_INF_F)) continue;
    const Key k = key_of(x, stop);
    const double t = total_of(k, b);
    if (!(t > -CUDART_INF) || t < on[K - 1]) continue;
    const int at = atomicAdd(&n_stop, 1);
    stop_key[at] = k;
    stop_at[at] = b;
  }
  __syncthreads();
  for (int i = tid; i < n_stop; i += JOIN_THREADS) {
    const Key k = stop_key[i];
    const int b = stop_at[i];
    const double t = total_of(k, b);
    auto in_front = [&](Key other, int c) {
      const double u = total_of(other, c);
      return u > t || (u == t && (c < b || (c == b && other > k)));
    };
    int place = 0, before = 0;
    for (int j = 0; j < n_stop; ++j) place += in_front(stop_key[j], stop_at[j]);
    for (int j = 0; j < K; ++j) before += on[j] > -CUDART_INF && in_front(keys[on_at[j]], on_at[j] / K);
    if (place + before < K) {
      a.ended_parents[r * K + place] = b;
      a.ended_tokens[r * K + place] = token_of(k);
      a.ended_scores[r * K + place] = (float)t;
    }
  }
  // ---- rows: a beam's best continuation stays in the beam's row ----
  if (warp == 0) {
    const bool live = lane < K && on[lane] > -CUDART_INF;
    const int parent = live ? on_at[lane] / K : -1 - lane;
    const unsigned same = __match_any_sync(0xffffffffu, parent);
    const bool stays = live && (same & ((1u << lane) - 1u)) == 0;
    const unsigned kept = __reduce_or_sync(0xffffffffu, stays ? 1u << parent : 0u);
    const unsigned moves = __ballot_sync(0xffffffffu, lane < K && !stays);
    if (lane < K) {
      int row = parent;
      if (!stays) {
        unsigned left = ~kept;
        for (int n = __popc(moves & ((1u << lane) - 1u)); n > 0; --n) left &= left - 1;
        row = __ffs(left) - 1;
      }
      a.parents[r * K + row] = live ? parent : -1;
      a.tokens[r * K + row] = live ? token_of(keys[on_at[lane]]) : 0;
      a.next_scores[r * K + row] = (float)on[lane];
    }
  }
}

size_t join_memory(int K, int S) { return (size_t)K * K * (8 + 8 + 8 + 4) + (size_t)K * S * (8 + 4); }
static_assert(MOST_BEAMS * (MOST_BEAMS * 28 + MOST_STOPS * 12) <= 40 * 1024, "the third launch's memory");

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
  const size_t memory = join_memory(K, S);
  jb::Launch join(dim3(R), dim3(JOIN_THREADS), memory, stream);
  return (int)cudaLaunchKernelEx(&join.c, beam_join_kernel, a);
}
