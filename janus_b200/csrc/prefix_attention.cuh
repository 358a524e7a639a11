// What the kernels of attention over a shared prefix have in common: a call's arguments, one row by one warp, and the join of
// partial results.
#pragma once
#include <math_constants.h>
#include <stdio.h>

#include "common.cuh"

namespace {

typedef __nv_bfloat16 bf16;

constexpr int PAGE = 64;
constexpr int SMS = 148;                 // multiprocessors
constexpr float LOG2E = 1.4426950408889634f;

// The sizes of a call and how it runs, as the caller hands them over (in one piece: passing them one by one cost the host more than a
// launch).  bfloat16: see jb_attention_prefix_bf16.  float32: `tiles` and `shared_per` are the rows of a block over the prefix and over
// own keys, `most` and `own_most` the ranges of both.
struct Sizes {
  int prefix_len, ld_table, width, T, n_pages, n_seqs, nh, nkv, hd, page_size, max_q_len, max_kv_len;
  int tiles, shared_per, most, own_tiles, own_ctas, fewest, own_most;
  float scale;
};
// ... and its tensors' places, in one piece as well.  scratch: see the entry points.
struct Tensors {
  const void *q, *k_cache, *v_cache;
  void* out;
  float* scratch;
  const int *prefix_pages, *block_table, *q_start, *kv_len, *positions;
};
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
// ranges of `per` places, the ranges that its tile is in.  Results over own keys begin at slot `most`.
struct Slots {
  int fixed, most, blocks, per, tile_tokens;
};
__device__ __forceinline__ int slots_of(const Slots& p, const Step& s, int token, int kvh) {
  if (p.fixed >= 0) return p.fixed;
  const int place = (token / p.tile_tokens * s.nkv + kvh) * p.blocks;
  return (place + p.blocks - 1) / p.per - place / p.per + 1;
}

// All partial results of a (token, query head) joined in the order of their slots, the prefix's first, then those over own keys:
// own_count[token][query head] of them (own_slots at most), or own_slots where that is null.  WARPS warps a row, each with every WARPS-th
// slot: four where there are few rows, which otherwise wait for one slot after another (464 rows of 35 slots: 19 us by one warp each),
// one where there are many.  Joined by the blocks that walk the own keys, one row after another, the wait took longer than the keys (48 sequences of up
// to 24 rows: 24 of 34 us).
template <typename E, int WARPS>
__global__ void __launch_bounds__(128) join_kernel(const E* __restrict__ q, const E* __restrict__ k_cache,
                                                   const E* __restrict__ v_cache, E* __restrict__ out,
                                                   const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                                                   const int* __restrict__ own_count, const Step s, const Slots parts, int own_slots) {
  __shared__ float4 red[WARPS > 1 ? WARPS * 64 : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = WARPS > 1 ? warp : 0;
  const int item = WARPS > 1 ? blockIdx.x : blockIdx.x * 4 + warp;
  const int t = item / s.nh, h = item - t * s.nh, kvh = h / (s.nh / s.nkv);
  const size_t all = (size_t)s.T * s.nh;
  const int shared = t < s.T ? slots_of(parts, s, t, kvh) : 0;
  const int total = s.q_start[s.n_seqs];   // (there since before the first of a call's launches, as all but partial results)
  jb::pdl_wait();
  jb::pdl_launch_dependents();
  if (t >= total || t >= s.T) return;
  auto place = [&](int i) { return (i < shared ? i : parts.most + i - shared) * all + item; };
  // How many results there are over own keys comes with the first results: what lies in places of none is not used.
  const int own = own_count ? own_count[item] : own_slots;
  float2 first = make_float2(-CUDART_INF_F, 0.0f);
  if (lane < shared + own_slots) first = part_ml[place(lane)];
  constexpr int EARLY = WARPS > 1 ? 2 : 0;   // (many rows hide one another's waits)
  float4 early[EARLY + 1][2];
#pragma unroll
  for (int i = 0; i < EARLY; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      early[i][e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (part + i * WARPS < shared && lane * 4 + 128 * e < s.hd)
        early[i][e] = *reinterpret_cast<const float4*>(part_o + place(part + i * WARPS) * s.hd + lane * 4 + 128 * e);
    }
  const int slots = shared + own;
  if (lane >= slots) first = make_float2(-CUDART_INF_F, 0.0f);
  float top = first.x, sum = 0.0f;
  for (int i = lane + 32; i < slots; i += 32) top = fmaxf(top, part_ml[place(i)].x);
  top = jb::warp_max(top);
  const float ref = top == -CUDART_INF_F ? 0.0f : top;
  float4 acc[2];
  acc[0] = acc[1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i0 = 0; i0 < slots; i0 += 32) {
    const float2 ml = i0 == 0 ? first : i0 + lane < slots ? part_ml[place(i0 + lane)] : make_float2(-CUDART_INF_F, 0.0f);
    const float mine = exp2f(ml.x - ref);
    sum = fmaf(mine, ml.y, sum);
    const int n = min(32, slots - i0);
    int j = part;
    if (i0 == 0) {
#pragma unroll
      for (int i = 0; i < EARLY; ++i)
        if (j < shared && j < n) {
          const float f = __shfl_sync(0xffffffffu, mine, j);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 v = early[i][e];
            acc[e].x = fmaf(f, v.x, acc[e].x), acc[e].y = fmaf(f, v.y, acc[e].y), acc[e].z = fmaf(f, v.z, acc[e].z), acc[e].w = fmaf(f, v.w, acc[e].w);
          }
          j += WARPS;
        }
    }
#pragma unroll 8
    for (; j < n; j += WARPS) {
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
  if constexpr (WARPS > 1) {
    red[warp * 64 + lane] = acc[0], red[warp * 64 + 32 + lane] = acc[1];
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 1; w < WARPS; ++w)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float4 v = red[w * 64 + 32 * e + lane];
        acc[e].x += v.x, acc[e].y += v.y, acc[e].z += v.z, acc[e].w += v.w;
      }
  }
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

// What a kernel needs set once: its shared memory's limit, and all of a multiprocessor's memory that can be shared as shared: kernels
// of unlike splits between cache and shared memory do not run on one multiprocessor together, and these are launched to overlap.
template <typename Kernel>
cudaError_t set_up(Kernel* kernel, int smem) {
  cudaError_t e = smem > 0 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) : cudaSuccess;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  return e;
}

template <typename E, int WARPS>
cudaError_t join_as(cudaStream_t stream, const E* q, const E* k, const E* v, E* out, const float* part_o, const float2* part_ml,
                    const int* own_count, const Step& s, const Slots& parts, int own_slots) {
  static bool configured = false;
  if (!configured) {
    cudaError_t e = set_up(join_kernel<E, WARPS>, 0);
    if (e != cudaSuccess) return e;
    configured = true;
  }
  const long long rows = (long long)s.T * s.nh;
  jb::Launch cfg(dim3((unsigned)(WARPS > 1 ? rows : (rows + 3) / 4)), dim3(128), 0, stream);
  return cudaLaunchKernelEx(&cfg.c, join_kernel<E, WARPS>, q, k, v, out, part_o, part_ml, own_count, s, parts, own_slots);
}
// (four warps a row up to what fits the multiprocessors at once, sixteen blocks each)
template <typename E>
cudaError_t join_go(cudaStream_t stream, const E* q, const E* k, const E* v, E* out, const float* part_o, const float2* part_ml,
                    const int* own_count, const Step& s, const Slots& parts, int own_slots) {
  return (long long)s.T * s.nh <= SMS * 16 ? join_as<E, 4>(stream, q, k, v, out, part_o, part_ml, own_count, s, parts, own_slots)
                                           : join_as<E, 1>(stream, q, k, v, out, part_o, part_ml, own_count, s, parts, own_slots);
}

}  // namespace
