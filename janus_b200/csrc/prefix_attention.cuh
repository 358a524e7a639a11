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

// Where the partial results over the prefix lie: slot i of a row is part_o [i][token][head][hd], part_ml [i][token][head].  How many
// slots a row has: `fixed`, or, where blocks cut the flat list of (tile of tile_tokens tokens, kv head) x `blocks` key blocks into
// ranges (the first `longer` of per + 1 places, the others of `per`), the ranges that its tile is in.  Results over own keys, where
// there are several, begin at slot `most`.
struct Slots {
  int fixed, most, blocks, per, longer, tile_tokens;
};
__device__ __forceinline__ int range_start(const Slots& p, int range) { return range * p.per + min(range, p.longer); }
__device__ __forceinline__ int range_of(const Slots& p, int place) {
  const int in_longer = p.longer * (p.per + 1);
  return place < in_longer ? place / (p.per + 1) : p.longer + (place - in_longer) / p.per;
}
__device__ __forceinline__ int slots_of(const Slots& p, const Step& s, int token, int kvh) {
  if (p.fixed >= 0) return p.fixed;
  const int place = (token / p.tile_tokens * s.nkv + kvh) * p.blocks;
  return range_of(p, place + p.blocks - 1) - range_of(p, place) + 1;
}

// One warp a (token, query head): all partial results joined in the order of their slots.
template <typename E>
__global__ void __launch_bounds__(128) join_kernel(const E* __restrict__ q, const E* __restrict__ k_cache,
                                                   const E* __restrict__ v_cache, E* __restrict__ out,
                                                   const float* __restrict__ part_o, const float2* __restrict__ part_ml, const Step s,
                                                   const Slots parts, int own_slots) {
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int t = item / s.nh, h = item % s.nh;
  if (t >= min(s.T, s.q_start[s.n_seqs])) return;
  const size_t all = (size_t)s.T * s.nh;
  const int shared = slots_of(parts, s, t, h / (s.nh / s.nkv)), slots = shared + own_slots;
  auto place = [&](int i) { return (i < shared ? i : parts.most + i - shared) * all + item; };
  float top = -CUDART_INF_F, sum = 0.0f;
  for (int i = lane; i < slots; i += 32) top = fmaxf(top, part_ml[place(i)].x);
  top = jb::warp_max(top);
  const float ref = top == -CUDART_INF_F ? 0.0f : top;
  float4 acc[2];
  acc[0] = acc[1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i0 = 0; i0 < slots; i0 += 32) {
    const float2 ml = i0 + lane < slots ? part_ml[place(i0 + lane)] : make_float2(-CUDART_INF_F, 0.0f);
    const float mine = exp2f(ml.x - ref);
    sum = fmaf(mine, ml.y, sum);
    const int n = min(32, slots - i0);
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const float f = __shfl_sync(0xffffffffu, mine, j);
      const float* row = part_o + place(i0 + j) * s.hd;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = lane * 4 + 128 * e;
        if (d < s.hd) {
          const float4 v = *reinterpret_cast<const float4*>(row + d);
          acc[e].x = fmaf(f, v.x, acc[e].x), acc[e].y = fmaf(f, v.y, acc[e].y), acc[e].z = fmaf(f, v.z, acc[e].z), acc[e].w = fmaf(f, v.w, acc[e].w);
        }
      }
    }
  }
  sum = jb::warp_sum(sum);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  bool finite = true;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int d = lane * 4 + 128 * e;
    if (d >= s.hd) continue;
    const float4 v = make_float4(acc[e].x * inv, acc[e].y * inv, acc[e].z * inv, acc[e].w * inv);
    store4(out + (size_t)item * s.hd + d, v);
    finite = finite && isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w);
  }
  if (__any_sync(0xffffffffu, !finite)) one_row(q, k_cache, v_cache, out, s, sequence_of(s, t), t, h);
}

// The last step of a block that holds WARPS partial results of each of `n_rows` rows in shared memory (red_o [WARPS][ROWS][ld],
// red_ml [WARPS][ROWS][2]): one more partial result in slot `put` of device memory (put >= 0), or joined with the prefix's and
// written, and a row that is not finite is made once more by itself.  Row r of the block is (token0 + (row0 + r) / G, query head
// kvh G + (row0 + r) % G).  `weights`: ROWS * parts.most floats of shared memory, `row_sums`: 2 ROWS floats.  All of a row's slots are
// asked for at once: one after another their latencies took longer than the sequence's own keys (18 slots, 64 sequences: 35 us).
template <typename E, int WARPS, int ROWS, int THREADS>
__device__ __forceinline__ void finish_rows(const E* q, const E* k_cache, const E* v_cache, E* out, float* part_o, float2* part_ml,
                                            const Step& s, const Slots& parts, const float* red_o, const float* red_ml, int ld,
                                            float* weights, float* row_sums, int n_rows, int row0, int token0, int seq, int kvh, int put) {
  const int G = s.nh / s.nkv, quads = s.hd / 4, lane = threadIdx.x & 31, most = put >= 0 ? 0 : parts.most;
  const size_t all = (size_t)s.T * s.nh;
  auto place_of = [&](int row) { return (size_t)(token0 + (row0 + row) / G) * s.nh + kvh * G + (row0 + row) % G; };
  // a warp a row: its maximum, its sum, and what each slot weighs
  for (int row = threadIdx.x >> 5; row < n_rows; row += THREADS / 32) {
    const size_t place = place_of(row);
    const int slots = most ? slots_of(parts, s, token0 + (row0 + row) / G, kvh) : 0;
    float top = -CUDART_INF_F, sum = 0.0f;
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, red_ml[2 * (w * ROWS + row)]);
    float2 ml[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {       // (at most 64 slots)
      ml[e] = lane + 32 * e < slots ? part_ml[(lane + 32 * e) * all + place] : make_float2(-CUDART_INF_F, 0.0f);
      top = fmaxf(top, ml[e].x);
    }
    top = jb::warp_max(top);
    const float ref = top == -CUDART_INF_F ? 0.0f : top;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float f = exp2f(ml[e].x - ref);
      if (lane + 32 * e < most) weights[row * most + lane + 32 * e] = lane + 32 * e < slots ? f : -1.0f;
      sum = fmaf(f, ml[e].y, sum);
    }
    sum = jb::warp_sum(sum);
    for (int w = 0; w < WARPS; ++w) sum = fmaf(exp2f(red_ml[2 * (w * ROWS + row)] - ref), red_ml[2 * (w * ROWS + row) + 1], sum);
    if (lane == 0) row_sums[2 * row] = top, row_sums[2 * row + 1] = sum;
  }
  __syncthreads();
  unsigned wrong = 0u;   // rows this thread found not finite, a bit for every row of its own
  int turn = 0;
  for (int idx = threadIdx.x; idx < n_rows * quads; idx += THREADS, ++turn) {
    const int row = idx / quads, d = idx % quads * 4;
    const size_t place = place_of(row);
    const float top = row_sums[2 * row], ref = top == -CUDART_INF_F ? 0.0f : top;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float f, const float4 v) {
      acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
    };
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int at = w * ROWS + row;
      add(exp2f(red_ml[2 * at] - ref), *reinterpret_cast<const float4*>(red_o + (size_t)at * ld + d));
    }
    if (put >= 0) {
      const size_t item = put * all + place;
      *reinterpret_cast<float4*>(part_o + item * s.hd + d) = acc;
      if (d == 0) part_ml[item] = make_float2(top, row_sums[2 * row + 1]);
      continue;
    }
    const float* from = part_o + place * s.hd + d;
#pragma unroll 8
    for (int i = 0; i < most; ++i) {
      const float f = weights[row * most + i];
      if (f >= 0.0f) add(f, *reinterpret_cast<const float4*>(from + i * all * s.hd));
    }
    const float sum = row_sums[2 * row + 1], inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
    store4(out + place * s.hd + d, acc);
    if (!(isfinite(acc.x) && isfinite(acc.y) && isfinite(acc.z) && isfinite(acc.w))) wrong |= 1u << min(turn, 31);
  }
  if (put >= 0) return;
  // (rare: nothing more is done where every number is finite)
  if (!__syncthreads_or(wrong != 0u)) return;
  for (int row = threadIdx.x; row < n_rows; row += THREADS) row_sums[2 * row] = 0.0f;
  __syncthreads();
  turn = 0;
  for (int idx = threadIdx.x; idx < n_rows * quads; idx += THREADS, ++turn)
    if (wrong >> min(turn, 31) & 1u) row_sums[2 * (idx / quads)] = 1.0f;
  __syncthreads();
  for (int row = threadIdx.x >> 5; row < n_rows; row += THREADS / 32)
    if (row_sums[2 * row] != 0.0f) one_row(q, k_cache, v_cache, out, s, seq, token0 + (row0 + row) / G, kvh * G + (row0 + row) % G);
}

}  // namespace
