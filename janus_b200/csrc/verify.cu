// Verification of drafted tokens against the target's logits, from given random numbers.
//
// Request b brings rows q_start[b] .. q_start[b + 1] - 1 of a step: the token it ended with and its drafts; the logits of a
// row judge the token of the next.  With w_v = exp((x_v - max) / T) and S the sum of w over a row:
//   a draft d is accepted while u q(d) S < w(d), q its probability under the drafting model (1 where drafts were looked up);
//   the row of the first refusal (or the last row) gives one more token: the lowest v whose cumulative weight C_v passes
//   u C, the weights being max(w / S - q, 0) after a refusal (w without d where drafts were looked up), else w.
// T = 0: a draft is accepted if it is the row's argmax (the lowest index of the largest), the token is the argmax.
#include <math_constants.h>
#include <stdio.h>

#include "common.cuh"

namespace {

constexpr int THREADS = 1024;

struct Row {
  float top, sum;
  int arg;
};

__device__ __forceinline__ float weight(float x, float top, float inv_heat) {
  if (!(x > -CUDART_INF_F)) return 0.0f;   // -inf, and what is not a number
  return x == top ? 1.0f : expf((x - top) * inv_heat);
}

__device__ Row row_stats(const float* x, int V, float inv_heat, float* scratch, int* scratch_i) {
  float top = -CUDART_INF_F;
  int arg = 0x7fffffff;
  for (int v = threadIdx.x; v < V; v += THREADS)
    if (x[v] > top) {
      top = x[v];
      arg = v;
    }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xffffffffu, top, o);
    const int i = __shfl_xor_sync(0xffffffffu, arg, o);
    if (t > top || (t == top && i < arg)) top = t, arg = i;
  }
  __syncthreads();
  if (lane == 0) scratch[warp] = top, scratch_i[warp] = arg;
  __syncthreads();
  top = scratch[0], arg = scratch_i[0];
  for (int w = 1; w < THREADS / 32; ++w)
    if (scratch[w] > top || (scratch[w] == top && scratch_i[w] < arg)) top = scratch[w], arg = scratch_i[w];
  float sum = 0.0f;
  for (int v = threadIdx.x; v < V; v += THREADS) sum += weight(x[v], top, inv_heat);
  __syncthreads();
  sum = jb::block_sum(sum, scratch);
  return Row{top, sum, arg == 0x7fffffff ? 0 : arg};
}

__global__ void __launch_bounds__(THREADS) verify_kernel(const float* __restrict__ logits, const int* __restrict__ tokens,
                                                         const int* __restrict__ q_start, const int* __restrict__ kv_len,
                                                         const float* __restrict__ u_accept, const float* __restrict__ u_draw,
                                                         const float* __restrict__ probs, int* __restrict__ accepted_out,
                                                         int* __restrict__ out, float* __restrict__ logprobs,
                                                         int* __restrict__ kept, int V, int width, int T, float heat) {
  __shared__ float scratch[40];
  __shared__ int scratch_i[32];
  __shared__ float s_sum[THREADS];
  __shared__ int s_token;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int lo = min(max(q_start[b], 0), T), hi = min(max(q_start[b + 1], lo), T), rows = min(hi - lo, width);
  const float inv_heat = heat > 0.0f ? 1.0f / heat : 1.0f;
  int* my = out + (size_t)b * width;
  float* lp = logprobs + (size_t)b * width;
  if (rows == 0) {
    for (int k = tid; k < width; k += THREADS) my[k] = -1, lp[k] = 0.0f;
    if (tid == 0) accepted_out[b] = 0, kept[b] = kv_len[b];
    return;
  }
  int accepted = 0;
  Row r;
  for (;; ++accepted) {
    const float* x = logits + (size_t)(lo + accepted) * V;
    r = row_stats(x, V, inv_heat, scratch, scratch_i);
    if (accepted == rows - 1) break;
    const int t = lo + accepted + 1, d = tokens[t];
    bool yes = d >= 0 && d < V;
    if (yes) {
      if (heat > 0.0f) {
        const float q = probs ? probs[(size_t)t * V + d] : 1.0f;
        yes = u_accept[t] * q * r.sum < weight(x[d], r.top, inv_heat);
      } else {
        yes = d == r.arg;
      }
    }
    if (!yes) break;
    if (tid == 0) my[accepted] = d, lp[accepted] = (x[d] - r.top) * inv_heat - logf(r.sum);
  }
  const float* x = logits + (size_t)(lo + accepted) * V;
  int token = r.arg;
  if (heat > 0.0f) {
    const bool refused = accepted < rows - 1;
    const int d = refused ? tokens[lo + accepted + 1] : -1;
    const float* q = refused && probs ? probs + (size_t)(lo + accepted + 1) * V : nullptr;
    const int per = (V + THREADS - 1) / THREADS, v0 = min(tid * per, V), v1 = min(v0 + per, V);
    for (int form = refused ? 0 : 1; form < 2; ++form) {
      auto mass = [&](int v) {
        const float w = weight(x[v], r.top, inv_heat);
        if (form == 1) return w;
        return q ? fmaxf(w / r.sum - q[v], 0.0f) : v == d ? 0.0f : w;
      };
      float mine = 0.0f;
      for (int v = v0; v < v1; ++v) mine += mass(v);
      s_sum[tid] = mine;
      __syncthreads();
      if (tid == 0) {
        float run = 0.0f;
        int last = -1;
        for (int i = 0; i < THREADS; ++i) {
          if (s_sum[i] > 0.0f) last = i;
          run += s_sum[i];
        }
        const float target = u_draw[b] * run;
        float before = 0.0f;
        int i = 0;
        while (i < last && !(target < before + s_sum[i])) before += s_sum[i++];
        s_token = -1;
        if (last >= 0) {
          const int a = min(i * per, V), e = min(a + per, V);
          for (int v = a; v < e; ++v) {
            const float w = mass(v);
            if (w > 0.0f) {
              before += w;
              s_token = v;
              if (target < before) break;
            }
          }
        }
      }
      __syncthreads();
      if (s_token >= 0) token = s_token;
      if (s_token >= 0) break;
    }
  }
  for (int k = accepted + 1 + tid; k < width; k += THREADS) my[k] = -1, lp[k] = 0.0f;
  if (tid == 0) {
    my[accepted] = token;
    lp[accepted] = (x[token] - r.top) * inv_heat - logf(r.sum);
    accepted_out[b] = accepted;
    kept[b] = kv_len[b] - (hi - lo - 1) + accepted;
  }
}

}  // namespace

JB_EXPORT int jb_verify_drafts(const float* logits, const int* tokens, const int* q_start, const int* kv_len, const float* u_accept,
                               const float* u_draw, const float* probs, int* accepted, int* out, float* logprobs, int* kept, int T,
                               int B, int V, int width, float heat, cudaStream_t stream) {
  if (B <= 0) return 0;
  JB_REFUSE(V <= 0 || width <= 0 || T < 0, "verify_drafts: %d rows of %d logits, %d tokens a request", T, V, width);
  verify_kernel<<<B, THREADS, 0, stream>>>(logits, tokens, q_start, kv_len, u_accept, u_draw, probs, accepted, out, logprobs, kept, V,
                                           width, T, heat);
  JB_CHECK_LAUNCH();
  return 0;
}
