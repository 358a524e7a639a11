// Verification of drafted tokens against the target's logits, from given random numbers.
//
// Request b brings rows q_start[b] .. q_start[b + 1] - 1 of a step: the token it ended with and its drafts; the logits of a
// row judge the token of the next.  With w_v = exp((x_v - max) / T) and S the sum of w over a row:
//   a draft d is accepted while u q(d) S < w(d), q its probability under the drafting model (1 where drafts were looked up);
//   the row of the first refusal (or the last row) gives one more token: the lowest v whose cumulative weight C_v passes
//   u C, the weights being max(w / S - q, 0) after a refusal (w without d where drafts were looked up), else w.
// T = 0: a draft is accepted if it is the row's argmax (the lowest index of the largest), the token is the argmax.
//
// Two launches, both bound by how fast rows come from memory.  `stats_kernel` reads every row once, in chunks of 8,192 logits that
// its threads hold in registers: a chunk's maximum, the sum of its weights against that maximum, its argmax.  `decide_kernel` has
// a cluster of up to 8 blocks a request: every block makes the request's decisions from the chunks' results (a few hundred numbers);
// where drafts of a drafting model were refused the blocks share out the pass over the row's weights and the draft's
// probabilities and tell one another the chunks' sums through distributed shared memory.  The chunk in which the drawn number falls
// is then read once more by the block that has it.  All sums are float32 in a fixed order.
//
// 256 requests of 1 to 5 drafts with probabilities, 128,256 logits: 100 us, the least 90 (587 MB at the measured 6,537 GB/s);
// stats_kernel 67 us of them at 6.8 TB/s, decide_kernel the rest: its passes over refused rows at 4 to 5 TB/s, behind 4.7 us of
// decisions.  64 requests over 32,000: 17.6 us for 32 MB, and one request 10.4: the second launch is a chain of waits (rows' results,
// the draw's chunk sums, the chunk, the token), which no bandwidth shortens.
#include <math_constants.h>
#include <stddef.h>
#include <stdio.h>

#include "common.cuh"

namespace {

constexpr int CHUNK = 8192;
constexpr int STATS_THREADS = 256, STATS_PER = CHUNK / STATS_THREADS;     // 32 logits a thread
constexpr int THREADS = 512, WARPS = THREADS / 32, PIECE = CHUNK / WARPS;   // a warp has 512 neighbouring logits of a chunk
constexpr int MAX_CLUSTER = 8;
constexpr float LOG2E = 1.4426950408889634f;

// 2^x by the special-function unit (2 ulp); -inf gives 0
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What is not a number counts as -inf.
__device__ __forceinline__ float number(float x) { return fmaxf(x, -CUDART_INF_F); }
// The weight of x (a number, or -inf) against a maximum; heat_log2 = log2(e) / T, finite.  A maximum of +inf or -inf: `weight`.
__device__ __forceinline__ float finite_weight(float x, float top, float heat_log2) { return fast_exp2((x - top) * heat_log2); }
__device__ __forceinline__ float weight(float x, float top, float heat_log2) {
  if (!(x > -CUDART_INF_F)) return 0.0f;
  return x == top ? 1.0f : finite_weight(x, top, heat_log2);
}

struct Chunk {
  float top, sum;
  int arg;
};

// (the larger value, of equal ones the lower index)
__device__ __forceinline__ void keep_first(float& top, int& arg, float t, int i) {
  if (t > top || (t == top && i < arg)) top = t, arg = i;
}

// ARGMAX: only where T = 0 asks for it (a third of the instructions a logit).
template <bool VECTORS, bool ARGMAX>
__global__ void __launch_bounds__(STATS_THREADS) stats_kernel(const float* __restrict__ logits, Chunk* __restrict__ stats, int V,
                                                              int chunks, float heat_log2) {
  __shared__ float s_top[STATS_THREADS / 32], s_sum[STATS_THREADS / 32];
  __shared__ int s_arg[STATS_THREADS / 32];
  jb::pdl_wait();
  jb::pdl_launch_dependents();
  const int row = blockIdx.x / chunks, chunk = blockIdx.x % chunks, v0 = chunk * CHUNK, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* x = logits + (size_t)row * V + v0;
  const int n = min(CHUNK, V - v0);
  float v[STATS_PER];
  if constexpr (VECTORS) {
#pragma unroll
    for (int i = 0; i < STATS_PER / 4; ++i) {
      const int at = (tid + STATS_THREADS * i) * 4;
      float4 t = make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
      if (at < n) t = __ldcs(reinterpret_cast<const float4*>(x + at));
      v[4 * i] = t.x, v[4 * i + 1] = t.y, v[4 * i + 2] = t.z, v[4 * i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < STATS_PER; ++i) {
      const int at = tid + STATS_THREADS * i;
      v[i] = at < n ? __ldcs(x + at) : -CUDART_INF_F;
    }
  }
  float top = -CUDART_INF_F;
  int arg = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < STATS_PER; ++i) {
    v[i] = number(v[i]);
    if constexpr (ARGMAX) {   // a thread's indices rise
      if (v[i] > top) top = v[i], arg = v0 + (VECTORS ? (tid + STATS_THREADS * (i / 4)) * 4 + i % 4 : tid + STATS_THREADS * i);
    } else {
      top = fmaxf(top, v[i]);
    }
  }
  if constexpr (ARGMAX) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float t = __shfl_xor_sync(0xffffffffu, top, o);
      const int i = __shfl_xor_sync(0xffffffffu, arg, o);
      keep_first(top, arg, t, i);
    }
    if (lane == 0) s_arg[warp] = arg;
  } else {
    top = jb::warp_max(top);
  }
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  top = s_top[0];
  if constexpr (ARGMAX) arg = s_arg[0];
#pragma unroll
  for (int w = 1; w < STATS_THREADS / 32; ++w) {
    if constexpr (ARGMAX) keep_first(top, arg, s_top[w], s_arg[w]);
    else top = fmaxf(top, s_top[w]);
  }
  float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (fabsf(top) < CUDART_INF_F) {
#pragma unroll
    for (int i = 0; i < STATS_PER; ++i) part[i & 3] += finite_weight(v[i], top, heat_log2);
  } else {
#pragma unroll
    for (int i = 0; i < STATS_PER; ++i) part[i & 3] += weight(v[i], top, heat_log2);
  }
  const float sum = jb::warp_sum((part[0] + part[1]) + (part[2] + part[3]));
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < STATS_THREADS / 32; ++w) all += s_sum[w];
    stats[blockIdx.x] = Chunk{top, all, arg};
  }
}

__device__ __forceinline__ int cluster_rank() {
  int r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ int cluster_size() {
  int n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The place of a variable of this block in the shared memory of block `rank` of the cluster
__device__ __forceinline__ uint32_t in_block(const void* p, int rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ void store_remote(uint32_t at, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}
__device__ __forceinline__ float warp_inclusive(float v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// What a token weighs in the draw: w (KEPT), w without token d (LOOKED_UP), what of p is more than q (REFUSED).
enum Form { KEPT, LOOKED_UP, REFUSED };
struct Draw {
  const float* x;
  const float* q;
  float top, inv_sum, heat_log2;
  int d, V;
  Form form;
  __device__ __forceinline__ float mass(int v, float xv, float qv) const {
    const float w = weight(number(xv), top, heat_log2);
    if (form == KEPT) return w;
    return form == LOOKED_UP ? (v == d ? 0.0f : w) : fmaxf(fmaf(w, inv_sum, -qv), 0.0f);
  }
  // four neighbouring tokens' logits, and their probabilities (REFUSED)
  __device__ __forceinline__ void load(int v0, bool vectors, float* xv, float* qv) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) xv[i] = -CUDART_INF_F, qv[i] = 0.0f;
    if (vectors) {
      if (v0 < V) *reinterpret_cast<float4*>(xv) = *reinterpret_cast<const float4*>(x + v0);
      if (v0 < V && form == REFUSED) *reinterpret_cast<float4*>(qv) = __ldcs(reinterpret_cast<const float4*>(q + v0));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (v0 + i < V) xv[i] = x[v0 + i];
        if (v0 + i < V && form == REFUSED) qv[i] = q[v0 + i];
      }
    }
  }
};

// The first of n masses (in order) whose running sum from `before` on passes `target`, or the last with any mass should rounding let
// none pass; -1: none has any.  start: the running sum in front of it; all: the sum of all.  By a whole warp, the same in every lane.
__device__ __forceinline__ int first_past(const float* mass, int n, float before, float target, float& start, float& all) {
  const int lane = threadIdx.x & 31;
  int pick = -1, last = -1;
  float run = before, last_start = before;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const float m = i0 + lane < n ? mass[i0 + lane] : 0.0f, up = run + warp_inclusive(m);
    const unsigned some = __ballot_sync(0xffffffffu, m > 0.0f), past = __ballot_sync(0xffffffffu, m > 0.0f && target < up);
    const float in_front = __shfl_up_sync(0xffffffffu, up, 1);
    const float mine = lane == 0 ? run : in_front;
    if (pick < 0 && past) {
      pick = i0 + __ffs(past) - 1;
      start = __shfl_sync(0xffffffffu, mine, __ffs(past) - 1);
    }
    if (some) {
      last = i0 + 31 - __clz(some);
      last_start = __shfl_sync(0xffffffffu, mine, 31 - __clz(some));
    }
    run = __shfl_sync(0xffffffffu, up, 31);
  }
  all = run;
  if (pick < 0) pick = last, start = last_start;
  return pick;
}

// A chunk's masses, 16 a thread (warp w has PIECE neighbouring tokens, in four runs of four a lane), and the warp's sum: the sums
// of runs in order.  run_end[k]: the warp's sum up to and with run k.
__device__ __forceinline__ float warp_masses(const Draw& draw, int chunk, bool vectors, float (&w)[16], float (&run_end)[4]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int v0 = chunk * CHUNK + warp * PIECE + lane * 4;
  float q[16];
#pragma unroll
  for (int k = 0; k < 4; ++k) draw.load(v0 + k * 128, vectors, w + 4 * k, q + 4 * k);   // all on their way before the first is looked at
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = draw.mass(v0 + i / 4 * 128 + i % 4, w[i], q[i]);
  float run = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    run += __shfl_sync(0xffffffffu, warp_inclusive(((w[4 * k] + w[4 * k + 1]) + w[4 * k + 2]) + w[4 * k + 3]), 31);
    run_end[k] = run;
  }
  return run;
}

__global__ void __launch_bounds__(THREADS, 2) decide_kernel(const float* __restrict__ logits, const Chunk* __restrict__ stats,
                                                         const int* __restrict__ tokens, const int* __restrict__ q_start,
                                                         const int* __restrict__ kv_len, const float* __restrict__ u_accept,
                                                         const float* __restrict__ u_draw, const float* __restrict__ probs,
                                                         int* __restrict__ accepted_out, int* __restrict__ out,
                                                         float* __restrict__ logprobs, int* __restrict__ kept, int V, int chunks, int width,
                                                         int T, float heat, float heat_log2, int vectors) {
  extern __shared__ float dyn[];
  float* chunk_sum = dyn;                                   // [chunks] masses of the drawn row's chunks
  float* warp_sums = chunk_sum + chunks;                    // [chunks][WARPS] ... of their warps' parts
  float* row_top = warp_sums + chunks * WARPS;              // [width] of the request's rows
  float* row_sum = row_top + width;                         // [width]
  int* row_arg = reinterpret_cast<int*>(row_sum + width);   // [width]
  int* row_yes = row_arg + width;                           // [width] the draft behind the row is accepted
  float* row_x = reinterpret_cast<float*>(row_yes + width); // [width] its logit
  __shared__ float s_warp[WARPS];
  __shared__ int s_token;
  const int size = cluster_size(), rank = cluster_rank(), b = blockIdx.x / size;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // What this launch reads was there before stats_kernel began (which has waited for it, where it ran), but for the chunks' results:
  // a row's draft and what is known of it are on their way while those are made.
  if (T == 0) jb::pdl_wait();
  const int lo = min(max(q_start[b], 0), T), hi = min(max(q_start[b + 1], lo), T), rows = min(hi - lo, width), cached = kv_len[b];
  const float u_token = u_draw[b];
  int* my = out + (size_t)b * width;
  float* lp = logprobs + (size_t)b * width;
  struct Draft {
    int d;
    float x, q, u;
  };
  auto draft_behind = [&](int r) {
    const int t = lo + r + 1, d = r + 1 < rows ? tokens[t] : -1;
    if (d < 0 || d >= V) return Draft{-1, 0.0f, 1.0f, 1.0f};
    return Draft{d, logits[(size_t)(lo + r) * V + d], probs && heat > 0.0f ? probs[(size_t)t * V + d] : 1.0f, u_accept[t]};
  };
  Draft draft = warp < rows ? draft_behind(warp) : Draft{};
  if (T > 0) jb::pdl_wait();
  jb::pdl_launch_dependents();
  if (rows == 0) {   // (the whole cluster)
    if (rank == 0) {
      for (int k = tid; k < width; k += THREADS) my[k] = -1, lp[k] = 0.0f;
      if (tid == 0) accepted_out[b] = 0, kept[b] = cached;
    }
    return;
  }
  // ---- a warp a row: its maximum and sum from its chunks', and the test of the draft behind it ----
  for (int r = warp; r < rows; r += WARPS) {
    const Chunk* c = stats + (size_t)(lo + r) * chunks;
    float top = -CUDART_INF_F, sum = 0.0f;
    int arg = 0x7fffffff;
    if (r != warp) draft = draft_behind(r);
    for (int i = lane; i < chunks; i += 32) keep_first(top, arg, c[i].top, c[i].arg);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float t = __shfl_xor_sync(0xffffffffu, top, o);
      const int i = __shfl_xor_sync(0xffffffffu, arg, o);
      keep_first(top, arg, t, i);
    }
    for (int i = lane; i < chunks; i += 32) sum = fmaf(c[i].sum, weight(c[i].top, top, heat_log2), sum);
    sum = jb::warp_sum(sum);
    if (arg == 0x7fffffff) arg = 0;
    if (lane == 0) {
      const bool yes = draft.d >= 0 && (heat > 0.0f ? draft.u * draft.q * sum < weight(draft.x, top, heat_log2) : draft.d == arg);
      row_top[r] = top, row_sum[r] = sum, row_arg[r] = arg, row_yes[r] = yes, row_x[r] = draft.x;
    }
  }
  if (tid == 0) s_token = -1;
  __syncthreads();
  int accepted = 0;
  while (accepted < rows - 1 && row_yes[accepted]) ++accepted;
  // ---- one more token, from row `accepted` ----
  int token = row_arg[accepted], writer = 0;
  if (heat > 0.0f) {
    const bool refused = accepted < rows - 1;
    const int next = lo + accepted + 1, d = refused ? tokens[next] : -1;
    const Chunk* c = stats + (size_t)(lo + accepted) * chunks;
    Draw draw{logits + (size_t)(lo + accepted) * V, probs ? probs + (size_t)min(next, T - 1) * V : nullptr, row_top[accepted],
              1.0f / row_sum[accepted], heat_log2, d, V, !refused ? KEPT : probs ? REFUSED : LOOKED_UP};
    const int c_begin = (int)((long long)rank * chunks / size), c_end = (int)((long long)(rank + 1) * chunks / size);
    const int d_chunk = draw.form == LOOKED_UP && d >= 0 && d < V ? d / CHUNK : -1;   // its sum is made anew, without d
    float w[16], run_end[4];
    auto chunk_mass = [&](int i) {   // by the whole block
      const float mine = warp_masses(draw, i, vectors, w, run_end);
      if (lane == 0) s_warp[warp] = mine;
      __syncthreads();
      float start, all;
      first_past(s_warp, WARPS, 0.0f, 0.0f, start, all);
      __syncthreads();
      return all;
    };
    // the chunks' masses, known to every block
    if (draw.form == REFUSED) {
      if (size > 1) cluster_sync();   // every block is there to be written to
      // (the warps do not wait for one another before the last chunk)
      for (int i = c_begin; i < c_end; ++i) {
        const float mine = warp_masses(draw, i, vectors, w, run_end);
        if (lane == 0) warp_sums[i * WARPS + warp] = mine;
      }
      __syncthreads();
      for (int i = c_begin + warp; i < c_end; i += WARPS) {
        float start, all;
        first_past(warp_sums + i * WARPS, WARPS, 0.0f, 0.0f, start, all);
        if (size == 1 && lane == 0) chunk_sum[i] = all;
        if (size > 1 && lane < size) store_remote(in_block(chunk_sum + i, lane), all);
      }
      if (size > 1) cluster_sync();
    }
    float total = 0.0f, before = 0.0f;
    for (int form = 0; form < 2; ++form) {
      if (form == 1 || draw.form != REFUSED) {
        const float again = d_chunk >= 0 && draw.form == LOOKED_UP ? chunk_mass(d_chunk) : 0.0f;
        for (int i = tid; i < chunks; i += THREADS)
          chunk_sum[i] = i == d_chunk && draw.form == LOOKED_UP ? again : c[i].sum * weight(c[i].top, draw.top, heat_log2);
      }
      __syncthreads();
      first_past(chunk_sum, chunks, 0.0f, 0.0f, before, total);
      if (total > 0.0f || draw.form == KEPT) break;
      draw.form = KEPT;   // nothing is left: from the row itself
      __syncthreads();
    }
    // the chunk where the drawn number falls
    const float target = u_token * total;
    const int pick = first_past(chunk_sum, chunks, 0.0f, target, before, total);
    if (pick >= 0) {
      writer = 0;
      while (!(pick < (int)((long long)(writer + 1) * chunks / size))) ++writer;
    }
    if (pick >= 0 && rank == writer) {
      const float mine = warp_masses(draw, pick, vectors, w, run_end);
      if (lane == 0) s_warp[warp] = mine;
      __syncthreads();
      float start, all;
      const int owner = first_past(s_warp, WARPS, before, target, start, all);
      if (warp == owner) {
        int hit = 0x7fffffff, last = -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float four = ((w[4 * k] + w[4 * k + 1]) + w[4 * k + 2]) + w[4 * k + 3];
          float sum = start + (k > 0 ? run_end[k > 0 ? k - 1 : 0] : 0.0f) + (warp_inclusive(four) - four);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int v = pick * CHUNK + warp * PIECE + k * 128 + lane * 4 + i;
            if (w[4 * k + i] > 0.0f) {
              sum += w[4 * k + i];
              last = v;
              if (target < sum) hit = min(hit, v);
            }
          }
        }
        hit = __reduce_min_sync(0xffffffffu, hit);
        last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) s_token = hit != 0x7fffffff ? hit : last;
      }
      __syncthreads();
      if (s_token >= 0) token = s_token;
    }
  }
  if (rank == writer) {
    for (int k = tid; k < width; k += THREADS) {
      int v = -1;
      float p = 0.0f;
      if (k <= accepted) {
        v = k < accepted ? tokens[lo + k + 1] : token;
        const float x = k < accepted ? row_x[k] : logits[(size_t)(lo + k) * V + v], gap = x == row_top[k] ? 0.0f : x - row_top[k];
        // (one over a temperature below 2.9e-39 is infinite, and 0 times it would not be a number)
        const float scaled = gap == 0.0f ? 0.0f : gap * (heat > 0.0f ? 1.0f / heat : 1.0f);
        p = row_sum[k] > 0.0f ? scaled - logf(row_sum[k]) : -CUDART_INF_F;
      }
      my[k] = v, lp[k] = p;
    }
    if (tid == 0) accepted_out[b] = accepted, kept[b] = cached - (hi - lo - 1) + accepted;
  }
}

struct Verify {
  const float* logits;
  const int *tokens, *q_start, *kv_len;
  const float *u_accept, *u_draw, *probs;   // probs: null where drafts were looked up
  int* accepted;
  int* out;
  float* logprobs;
  int* kept;
  void* stats;            // scratch of 3 floats a row and chunk of 8,192 logits
  int T, B, V, width;
  float heat;
};
}  // namespace

// given: a Verify in host memory.  The launch of decide_kernel is by clusters.
JB_EXPORT int jb_verify_drafts(const void* given, cudaStream_t stream) {
  static_assert(offsetof(Verify, heat) == 12 * 8 + 4 * 4, "as the caller packs it");
  const Verify& g = *(const Verify*)given;
  const float *logits = g.logits, *u_accept = g.u_accept, *u_draw = g.u_draw, *probs = g.probs;
  const int T = g.T, B = g.B, V = g.V, width = g.width;
  const float heat = g.heat;
  void* stats = g.stats;
  if (B <= 0) return 0;
  JB_REFUSE(V <= 0 || width <= 0 || T < 0, "verify_drafts: %d rows of %d logits, %d tokens a request", T, V, width);
  const int chunks = (V + CHUNK - 1) / CHUNK;
  const size_t smem = ((size_t)chunks * (1 + WARPS) + 5 * (size_t)width) * sizeof(float);
  JB_REFUSE(smem > 48 * 1024, "verify_drafts: %d tokens a request over a vocabulary of %d", width, V);
  JB_REFUSE((long long)T * chunks > 0x7fffffffll || (long long)B * MAX_CLUSTER > 0x7fffffffll, "verify_drafts: %d rows of %d logits", T, V);
  const float heat_log2 = heat > 0.0f ? fminf(LOG2E / heat, 1e30f) : LOG2E;   // (finite: 0 times it is 0)
  const bool vectors = V % 4 == 0 && (((uintptr_t)logits | (uintptr_t)probs) & 15) == 0;
  cudaError_t e = cudaSuccess;
  if (T > 0) {
    jb::Launch cfg(dim3(T * chunks), dim3(STATS_THREADS), 0, stream);
    e = cudaLaunchKernelEx(&cfg.c, heat > 0.0f ? (vectors ? stats_kernel<true, false> : stats_kernel<false, false>)
                                              : (vectors ? stats_kernel<true, true> : stats_kernel<false, true>), logits, (Chunk*)stats, V, chunks, heat_log2);
    if (e != cudaSuccess) return (int)e;
  }
  // Blocks a request: as many as run at once (two a multiprocessor), twice.  A block more takes its share of a row's chunks, but makes all
  // of the request's decisions too.  One where no row is passed over, drafts having been looked up (221 requests: 49 us, 58 by two each).
  int size = probs && heat > 0.0f ? 4 * 148 / B : 1;
  size = size < 1 ? 1 : size > MAX_CLUSTER ? MAX_CLUSTER : size;
  if (size > chunks) size = chunks;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(B * size), cfg.blockDim = dim3(THREADS), cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  cfg.attrs = attr, cfg.numAttrs = jb::pdl_enabled() ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, decide_kernel, logits, (const Chunk*)stats, g.tokens, g.q_start, g.kv_len, u_accept, u_draw, probs,
                                 g.accepted, g.out, g.logprobs, g.kept, V, chunks, width, T, heat, heat_log2, (int)vectors);
}
