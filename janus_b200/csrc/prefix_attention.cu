// Attention of a step whose sequences share a prefix: every query sees the prefix's keys and its own sequence's, up to its
// own position.  Key i of the prefix lies in page prefix_pages[i / 64], key prefix_len + i of sequence b in page
// block_table[b][i / 64].  softmax(q K^T scale) V over both together; kv head of query head h is floor(h nkv / nh).
#include <math_constants.h>
#include <stdio.h>

#include "common.cuh"

namespace {

constexpr int PAGE = 64;
constexpr float LOG2E = 1.4426950408889634f;

// One warp a (token, query head); a lane has every 32nd number of the head.
template <typename E>
__global__ void __launch_bounds__(128) prefix_attention_kernel(
    const E* __restrict__ q, const E* __restrict__ k_cache, const E* __restrict__ v_cache, E* __restrict__ out,
    const int* __restrict__ prefix_pages, int prefix_len, const int* __restrict__ block_table, int ld_table,
    const int* __restrict__ q_start, const int* __restrict__ kv_len, const int* __restrict__ positions, int T, int n_seqs, int nh,
    int nkv, int hd, float scale_log2) {
  const int warp = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int t = warp / nh, h = warp % nh;
  if (t >= T || t >= q_start[n_seqs]) return;
  int lo = 0, hi = n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (q_start[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int kvh = h / (nh / nkv), pos = positions[t], last = min(pos, kv_len[lo] - 1);
  float qr[8], o[8], m = -CUDART_INF_F, l = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    qr[i] = d < hd ? jb::to_f32(q[((size_t)t * nh + h) * hd + d]) * scale_log2 : 0.0f;
    o[i] = 0.0f;
  }
  for (int p = 0; p <= last; ++p) {
    const int i0 = p < prefix_len ? p : p - prefix_len;
    const int page = p < prefix_len ? prefix_pages[i0 / PAGE] : block_table[(size_t)lo * ld_table + i0 / PAGE];
    const size_t row = (((size_t)max(page, 0) * nkv + kvh) * PAGE + i0 % PAGE) * hd;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < hd) s = fmaf(qr[i], jb::to_f32(k_cache[row + lane + 32 * i]), s);
    s = jb::warp_sum(s);
    const float m_new = fmaxf(m, s), ref = m_new == -CUDART_INF_F ? 0.0f : m_new;
    const float corr = exp2f(m - ref), w = exp2f(s - ref);
    m = m_new;
    l = l * corr + w;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < hd) o[i] = o[i] * corr + w * jb::to_f32(v_cache[row + lane + 32 * i]);
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < hd) out[((size_t)t * nh + h) * hd + lane + 32 * i] = jb::from_f32<E>(o[i] * inv);
}

}  // namespace

JB_EXPORT int jb_attention_prefix(const void* q, const void* k_cache, const void* v_cache, void* out, int dtype,
                                  const int* prefix_pages, int prefix_len, const int* block_table, int ld_table,
                                  const int* q_start, const int* kv_len, const int* positions, int T, int n_seqs, int nh, int nkv,
                                  int hd, int page_size, float scale, cudaStream_t stream) {
  if (T <= 0 || n_seqs <= 0) return 0;
  JB_REFUSE(page_size != PAGE, "attention_prefix: page size %d (need %d)", page_size, PAGE);
  JB_REFUSE(nkv <= 0 || nh % nkv != 0, "attention_prefix: %d heads are not a multiple of %d kv heads", nh, nkv);
  JB_REFUSE(hd <= 0 || hd > 256, "attention_prefix: head size %d", hd);
  const unsigned blocks = (unsigned)(((long long)T * nh + 3) / 4);
  if (dtype == JB_BF16)
    prefix_attention_kernel<__nv_bfloat16><<<blocks, 128, 0, stream>>>(
        (const __nv_bfloat16*)q, (const __nv_bfloat16*)k_cache, (const __nv_bfloat16*)v_cache, (__nv_bfloat16*)out, prefix_pages,
        prefix_len, block_table, ld_table, q_start, kv_len, positions, T, n_seqs, nh, nkv, hd, scale * LOG2E);
  else if (dtype == JB_F32)
    prefix_attention_kernel<float><<<blocks, 128, 0, stream>>>((const float*)q, (const float*)k_cache, (const float*)v_cache, (float*)out,
                                                               prefix_pages, prefix_len, block_table, ld_table, q_start, kv_len,
                                                               positions, T, n_seqs, nh, nkv, hd, scale * LOG2E);
  else
    return JB_ERR_BAD_DTYPE;
  JB_CHECK_LAUNCH();
  return 0;
}
