// What the kernels of attention over a shared prefix have in common: a call's arguments, one row by one warp, and the join of
// partial results.
#pragma once
#include <math_constants.h>
#include <stdio.h>

#include "common.cuh"

namespace {

typedef __nv_bfloat16 bf16;

constexpr int PAGE = 64;
constexpr float LOG2E = 1.4426950408889634f;

// What every kernel of a call knows.
struct Step {
  const int* prefix_pages;
  const int* table;       // [n_seqs] rows of ld_table pages
  const int* q_start;
  const int* kv_len;
  const int* positions;
  int prefix_len, ld_table, width, T, n_seqs, nh, nkv, hd;
  float scale_log2;
};

// ---------------------------------------------------------------------------
// One (token, query head) by one warp, a lane with every 32nd number of the head: keys one after another, nothing but the
// keys that the token sees.  The float32 engine's form, and where a tiled kernel's result is not finite: a masked key weighs 0
// there, and 0 times what is not a number in a masked value's place would show.
// ---------------------------------------------------------------------------
template <typename E>
__device__ __noinline__ void one_row(const E* __restrict__ q, const E* __restrict__ k_cache, const E* __restrict__ v_cache,
                                     E* __restrict__ out, const Step& s, int seq, int t, int h) {
  const int lane = threadIdx.x & 31;
  const int kvh = h / (s.nh / s.nkv), last = min(min(s.positions[t], s.kv_len[seq] - 1), s.prefix_len + s.width * PAGE - 1);
  float qr[8], o[8], m = -CUDART_INF_F, l = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    qr[i] = d < s.hd ? jb::to_f32(q[((size_t)t * s.nh + h) * s.hd + d]) * s.scale_log2 : 0.0f;
    o[i] = 0.0f;
  }
  for (int p = 0; p <= last; ++p) {
    const int i0 = p < s.prefix_len ? p : p - s.prefix_len;
    const int page = p < s.prefix_len ? s.prefix_pages[i0 / PAGE] : s.table[(size_t)seq * s.ld_table + i0 / PAGE];
    const size_t row = (((size_t)max(page, 0) * s.nkv + kvh) * PAGE + i0 % PAGE) * s.hd;
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < s.hd) x = fmaf(qr[i], jb::to_f32(k_cache[row + lane + 32 * i]), x);
    x = jb::warp_sum(x);
    const float m_new = fmaxf(m, x), ref = m_new == -CUDART_INF_F ? 0.0f : m_new;
    const float corr = exp2f(m - ref), w = exp2f(x - ref);
    m = m_new;
    l = l * corr + w;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < s.hd) o[i] = o[i] * corr + w * jb::to_f32(v_cache[row + lane + 32 * i]);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < s.hd) out[((size_t)t * s.nh + h) * s.hd + lane + 32 * i] = jb::from_f32<E>(o[i] * inv);
}

__device__ __forceinline__ int sequence_of(const Step& s, int t) {
  int lo = 0, hi = s.n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (s.q_start[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ void store4(bf16* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }

// One warp a (token, query head): all partial results joined in the order of their slots.
template <typename E>
__global__ void __launch_bounds__(128) join_kernel(const E* __restrict__ q, const E* __restrict__ k_cache,
                                                   const E* __restrict__ v_cache, E* __restrict__ out,
                                                   const float* __restrict__ part_o, const float2* __restrict__ part_ml, const Step s,
                                                   int slots) {
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int t = item / s.nh, h = item % s.nh;
  if (t >= min(s.T, s.q_start[s.n_seqs])) return;
  const size_t all = (size_t)s.T * s.nh;
  float top = -CUDART_INF_F;
  for (int i = 0; i < slots; ++i) top = fmaxf(top, part_ml[i * all + item].x);
  const float ref = top == -CUDART_INF_F ? 0.0f : top;
  bool finite = true;
  for (int d = lane * 4; d < s.hd; d += 128) {
    float sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i = 0; i < slots; ++i) {
      const float2 ml = part_ml[i * all + item];
      const float f = exp2f(ml.x - ref);
      const float4 v = *reinterpret_cast<const float4*>(part_o + (i * all + item) * s.hd + d);
      sum = fmaf(f, ml.y, sum);
      acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
    store4(out + (size_t)item * s.hd + d, acc);
    finite = finite && isfinite(acc.x) && isfinite(acc.y) && isfinite(acc.z) && isfinite(acc.w);
  }
  if (__any_sync(0xffffffffu, !finite)) one_row(q, k_cache, v_cache, out, s, sequence_of(s, t), t, h);
}

// The last step of a block that holds WARPS partial results of each of `n_rows` rows in shared memory (red_o [WARPS][rows][ld],
// red_ml [WARPS][rows][2]): with own_slots > 1 they become one more partial result in device memory; else they are joined with the
// prefix's (their slots come first) and written, and a row that is not finite is made once more by itself.  Row r of the block is
// (token0 + (row0 + r) / G, query head kvh G + (row0 + r) % G).  `not_finite`: n_rows ints, zero.
template <typename E, int WARPS, int ROWS, int THREADS>
__device__ __forceinline__ void finish_rows(const E* q, const E* k_cache, const E* v_cache, E* out, float* part_o, float2* part_ml,
                                            const Step& s, const float* red_o, const float* red_ml, int ld, int* not_finite, int n_rows,
                                            int row0, int token0, int seq, int kvh, int prefix_slots, int own_slots, int split) {
  const int G = s.nh / s.nkv, quads = s.hd / 4;
  const size_t all = (size_t)s.T * s.nh;
  for (int idx = threadIdx.x; idx < n_rows * quads; idx += THREADS) {
    const int row = idx / quads, d = idx % quads * 4, rr = row0 + row;
    const size_t place = (size_t)(token0 + rr / G) * s.nh + kvh * G + rr % G;
    float top = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, red_ml[2 * (w * ROWS + row)]);
    if (own_slots == 1)
      for (int i = 0; i < prefix_slots; ++i) top = fmaxf(top, part_ml[i * all + place].x);
    const float ref = top == -CUDART_INF_F ? 0.0f : top;
    float sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float f, float li, const float4 v) {
      sum = fmaf(f, li, sum);
      acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
    };
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int at = w * ROWS + row;
      add(exp2f(red_ml[2 * at] - ref), red_ml[2 * at + 1], *reinterpret_cast<const float4*>(red_o + (size_t)at * ld + d));
    }
    if (own_slots > 1) {
      const size_t item = (prefix_slots + split) * all + place;
      *reinterpret_cast<float4*>(part_o + item * s.hd + d) = acc;
      if (d == 0) part_ml[item] = make_float2(top, sum);
      continue;
    }
    for (int i = 0; i < prefix_slots; ++i) {
      const size_t item = i * all + place;
      const float2 ml = part_ml[item];
      add(exp2f(ml.x - ref), ml.y, *reinterpret_cast<const float4*>(part_o + item * s.hd + d));
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
    store4(out + place * s.hd + d, acc);
    if (!(isfinite(acc.x) && isfinite(acc.y) && isfinite(acc.z) && isfinite(acc.w))) not_finite[row] = 1;
  }
  if (own_slots > 1) return;
  __syncthreads();
  for (int row = threadIdx.x >> 5; row < n_rows; row += THREADS / 32)
    if (not_finite[row]) one_row(q, k_cache, v_cache, out, s, seq, token0 + (row0 + row) / G, kvh * G + (row0 + row) % G);
}

}  // namespace
