// Attention of a step whose sequences share a prefix (see prefix_attention.cu) in true float32, without tensor cores.
//
// The same split: the prefix's keys in ranges for the rows of all sequences together, each sequence's own pages, partial results
// joined.  A block has 16 RR rows (token, query head of one kv head) and walks pages of 64 keys.  Thread (y, x) of 16 x 16 has RR
// rows and keys x, x + 16, .. of the scores, then the same rows and numbers 4 x .. 4 x + 3, 64 further, .. of the weighted values:
// products of RR x 4 out of shared memory, two multiply-adds an instruction.  A page's values are on their way during its scores.  Head
// sizes that are no multiple of 4 go row by row.
//
// Bound by the multiply-adds and the reads of shared memory beside them: 60 tokens, 16 heads over 4 of 128, behind 6,000 with up to 540
// own: 112 us, 41 of them the multiply-adds at their full rate; 29 tokens behind 2,050, a page a block: 41 us, of which 8 (the
// rest: loads in front of the products, 33 partial results a row, three launches).
#include "prefix_attention.cuh"

namespace {

__global__ void __launch_bounds__(128) rows_f32_kernel(const float* __restrict__ q, const float* __restrict__ k_cache,
                                                       const float* __restrict__ v_cache, float* __restrict__ out, const Step s) {
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  const int warp = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = warp / s.nh, h = warp % s.nh;
  if (t >= s.T || t >= s.q_start[s.n_seqs]) return;
  one_row(q, k_cache, v_cache, out, s, sequence_of(s, t), t, h);
}

constexpr int THREADS = 256;

__device__ __forceinline__ void cp_async16(float* dst, const float* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int HDC, int RR>
struct Tile {
  static constexpr int ROWS = 16 * RR, LD = HDC + 4, LD_P = PAGE + 4;
  // queries, keys, values.  The weights take the keys' place once the scores are made, the rows' results the place of keys and values
  // at the end.  Two blocks share a multiprocessor (heads of up to 128 numbers), and one's products hide the other's loads.
  static constexpr int FLOATS = ROWS * LD + PAGE * LD + PAGE * LD;
  static constexpr int SMEM = FLOATS * 4, BLOCKS = HDC <= 128 ? 2 : 1;
  static_assert(ROWS * LD_P <= PAGE * LD, "the weights' place");
  static_assert(SMEM <= 232448 && ROWS <= PAGE, "shared memory of one block");
};

// OWN: the rows of one sequence over its own pages.  Else the rows of all sequences over a range of the prefix's pages.
template <int HDC, int RR, bool OWN>
__global__ void __launch_bounds__(THREADS, (Tile<HDC, RR>::BLOCKS)) tile_f32_kernel(const float* __restrict__ q, const float* __restrict__ k_cache,
                                                           const float* __restrict__ v_cache, float* __restrict__ part_o,
                                                           float2* __restrict__ part_ml, const Step s,
                                                           const Slots parts, int own_slots, int row_blocks) {
  typedef Tile<HDC, RR> C;
  extern __shared__ __align__(16) float smem[];
  __shared__ float red_ml[2 * C::ROWS];
  float *q_s = smem, *k_s = q_s + C::ROWS * C::LD, *v_s = k_s + PAGE * C::LD, *p_s = k_s;
  const int G = s.nh / s.nkv, hd = s.hd, tid = threadIdx.x, x = tid & 15, y = tid >> 4;
  const int prefix_slots = parts.fixed;
  // (a launch over own keys right behind the one over the prefix finds everything in its place but that one's results, which it
  // does not read)
  if (!OWN || prefix_slots == 0) jb::pdl_wait();
  jb::pdl_launch_dependents();
  int seq = 0, kvh, split = blockIdx.z, token0 = 0, row0, n_rows, first_pos = 0, p_begin, p_end;
  const int* pages;
  if constexpr (OWN) {
    seq = blockIdx.x, kvh = blockIdx.y / row_blocks, row0 = blockIdx.y % row_blocks * C::ROWS;
    token0 = s.q_start[seq];
    const int q_len = s.q_start[seq + 1] - token0;
    n_rows = min(C::ROWS, q_len * G - row0);
    first_pos = s.kv_len[seq] - q_len - s.prefix_len;          // among the own keys
    const int see = n_rows > 0 ? first_pos + (row0 + n_rows - 1) / G + 1 : 0;
    const int n = min(see > 0 ? (see + PAGE - 1) / PAGE : 0, s.width);
    p_begin = (int)((long long)split * n / own_slots), p_end = (int)((long long)(split + 1) * n / own_slots);
    pages = s.table + (size_t)seq * s.ld_table;
  } else {
    kvh = blockIdx.x, row0 = blockIdx.y * C::ROWS;
    n_rows = min(C::ROWS, min(s.T, max(s.q_start[s.n_seqs], 0)) * G - row0);
    const int n = (s.prefix_len + PAGE - 1) / PAGE;
    p_begin = (int)((long long)split * n / prefix_slots), p_end = (int)((long long)(split + 1) * n / prefix_slots);
    pages = s.prefix_pages;
  }
  if (!OWN && n_rows <= 0) return;
  if (n_rows <= 0) p_end = p_begin;
  const int quads = hd / 4;
  auto load = [&](float* dst, const float* cache, int p) {
    const float* src = cache + ((size_t)max(pages[p], 0) * s.nkv + kvh) * PAGE * hd;
    for (int i = tid; i < PAGE * quads; i += THREADS) cp_async16(dst + i / quads * C::LD + i % quads * 4, src + (size_t)i * 4);
    cp_async_commit();
  };
  if (p_begin < p_end) {
    for (int i = tid; i < C::ROWS * quads; i += THREADS) {
      const int r = i / quads, rr = row0 + r;
      if (r < n_rows) cp_async16(q_s + r * C::LD + i % quads * 4, q + ((size_t)(token0 + rr / G) * s.nh + kvh * G + rr % G) * hd + i % quads * 4);
      else *reinterpret_cast<float4*>(q_s + r * C::LD + i % quads * 4) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    load(k_s, k_cache, p_begin);
    load(v_s, v_cache, p_begin);
  }
  int see[RR];
  float m[RR], l[RR];
  jb::Pair o[RR][HDC / 32];
#pragma unroll
  for (int r = 0; r < RR; ++r) {
    const int rr = row0 + y * RR + r;
    see[r] = 0;
    if (y * RR + r < n_rows) see[r] = OWN ? first_pos + rr / G + 1 : min(s.positions[rr / G] + 1, s.prefix_len);
    m[r] = -CUDART_INF_F, l[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < HDC / 32; ++i) o[r][i] = 0ull;
  }
  for (int p = p_begin; p < p_end; ++p) {
    cp_async_wait<1>();          // the page's keys (and the queries); its values may still be on their way
    __syncthreads();
    jb::Pair acc[RR][4];
#pragma unroll
    for (int r = 0; r < RR; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[r][k] = 0ull;
#pragma unroll 4
    for (int d = 0; d < hd; d += 4) {
      ulonglong2 kv[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) kv[k] = *reinterpret_cast<const ulonglong2*>(k_s + (x + 16 * k) * C::LD + d);
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        const ulonglong2 qv = *reinterpret_cast<const ulonglong2*>(q_s + (y * RR + r) * C::LD + d);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[r][k] = jb::fma2(qv.y, kv[k].y, jb::fma2(qv.x, kv[k].x, acc[r][k]));
      }
    }
    __syncthreads();             // the keys have been read
    float corr[RR];
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      float sc[4], top = -CUDART_INF_F;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        sc[k] = p * PAGE + x + 16 * k < see[r] ? (jb::lo(acc[r][k]) + jb::hi(acc[r][k])) * s.scale_log2 : -CUDART_INF_F;
        top = fmaxf(top, sc[k]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float m_new = fmaxf(m[r], top), ref = m_new == -CUDART_INF_F ? 0.0f : m_new;
      corr[r] = exp2f(m[r] - ref);
      m[r] = m_new;
      l[r] *= corr[r];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float w = exp2f(sc[k] - ref);
        l[r] += w;
        p_s[(y * RR + r) * C::LD_P + x + 16 * k] = w;
      }
#pragma unroll
      for (int i = 0; i < HDC / 32; ++i) o[r][i] = jb::mul2(o[r][i], jb::pair(corr[r], corr[r]));
    }
    cp_async_wait<0>();          // the page's values
    __syncthreads();
#pragma unroll 2
    for (int k = 0; k < PAGE; k += 4) {
      float4 w[RR];
#pragma unroll
      for (int r = 0; r < RR; ++r) w[r] = *reinterpret_cast<const float4*>(p_s + (y * RR + r) * C::LD_P + k);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < HDC / 64; ++i) {
          if (4 * x + 64 * i >= hd) break;
          const ulonglong2 vv = *reinterpret_cast<const ulonglong2*>(v_s + (k + j) * C::LD + 4 * x + 64 * i);
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            const float f = j == 0 ? w[r].x : j == 1 ? w[r].y : j == 2 ? w[r].z : w[r].w;
            const jb::Pair f2 = jb::pair(f, f);
            o[r][2 * i] = jb::fma2(f2, vv.x, o[r][2 * i]);
            o[r][2 * i + 1] = jb::fma2(f2, vv.y, o[r][2 * i + 1]);
          }
        }
      }
    }
    __syncthreads();
    if (p + 1 < p_end) {
      load(k_s, k_cache, p + 1);
      load(v_s, v_cache, p + 1);
    }
  }
  __syncthreads();
  float* red_o = k_s;
#pragma unroll
  for (int r = 0; r < RR; ++r) {
    const int row = y * RR + r;
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
    if (x == 0) red_ml[2 * row] = m[r], red_ml[2 * row + 1] = l[r];
#pragma unroll
    for (int i = 0; i < HDC / 64; ++i) {
      ulonglong2 v;
      v.x = o[r][2 * i], v.y = o[r][2 * i + 1];
      if (4 * x + 64 * i < hd) *reinterpret_cast<ulonglong2*>(red_o + row * C::LD + 4 * x + 64 * i) = v;
    }
  }
  __syncthreads();
  const int slot = OWN ? parts.most + split : split;
  for (int i = tid; i < n_rows * quads; i += THREADS) {
    const int r = i / quads, d = i % quads * 4, rr = row0 + r;
    const size_t item = (size_t)slot * s.T * s.nh + (size_t)(token0 + rr / G) * s.nh + kvh * G + rr % G;
    *reinterpret_cast<float4*>(part_o + item * hd + d) = *reinterpret_cast<const float4*>(red_o + r * C::LD + d);
    if (d == 0) part_ml[item] = make_float2(red_ml[2 * r], red_ml[2 * r + 1]);
  }
  // (who waits for this launch has to have waited for the one before it: one block sees to that)
  if (OWN && prefix_slots > 0 && blockIdx.x + blockIdx.y + blockIdx.z == 0) jb::pdl_wait();
}

template <int HDC, int RR, bool OWN>
cudaError_t go(dim3 grid, cudaStream_t stream, const float* q, const float* k, const float* v, float* part_o, float2* part_ml,
               const Step& s, const Slots& parts, int own_slots, int row_blocks) {
  typedef Tile<HDC, RR> C;
  static bool configured = false;
  if (!configured) {
    cudaError_t e = set_up(tile_f32_kernel<HDC, RR, OWN>, C::SMEM);
    if (e != cudaSuccess) return e;
    configured = true;
  }
  jb::Launch cfg(grid, dim3(THREADS), C::SMEM, stream);
  return cudaLaunchKernelEx(&cfg.c, tile_f32_kernel<HDC, RR, OWN>, q, k, v, part_o, part_ml, s, parts, own_slots, row_blocks);
}
template <bool OWN>
cudaError_t pick(int hd, int rows, dim3 grid, cudaStream_t stream, const float* q, const float* k, const float* v, float* part_o,
                 float2* part_ml, const Step& s, const Slots& parts, int own_slots, int row_blocks) {
#define JB_GO(HDC)                                                                                                              \
  return rows == 16 ? go<HDC, 1, OWN>(grid, stream, q, k, v, part_o, part_ml, s, parts, own_slots, row_blocks)       \
                    : go<HDC, 4, OWN>(grid, stream, q, k, v, part_o, part_ml, s, parts, own_slots, row_blocks)
  if (hd > 128) JB_GO(256);
  if (hd > 64) JB_GO(128);
  JB_GO(64);
#undef JB_GO
}

}  // namespace

// q, out [T, nh hd], caches [n_pages, nkv, 64, hd], all float32.  splits: ranges of the prefix (0: there is none), own_slots: ranges
// of a sequence's own keys; rows, own_rows: rows of a block over the prefix and over own keys, 16 or 64; scratch: floats
// [splits + own_slots][T][nh][hd], then [..][T][nh][2].  Head sizes that are no multiple of 4 use none of these.
// tensors, sizes: host memory, see Tensors and Sizes.
JB_EXPORT int jb_attention_prefix_f32(const void* tensors, const void* sizes, cudaStream_t stream) {
  const Tensors& t = *(const Tensors*)tensors;
  const Sizes& z = *(const Sizes*)sizes;
  const void *q = t.q, *k_cache = t.k_cache, *v_cache = t.v_cache;
  void* out = t.out;
  float* scratch = t.scratch;
  const int prefix_len = z.prefix_len, T = z.T, n_seqs = z.n_seqs, nh = z.nh, nkv = z.nkv, hd = z.hd, page_size = z.page_size;
  const int max_q_len = z.max_q_len, rows = z.tiles, own_rows = z.shared_per, splits = z.most, own_slots = z.own_most;
  if (T <= 0 || n_seqs <= 0 || max_q_len <= 0) return 0;
  JB_REFUSE(page_size != PAGE, "attention_prefix: page size %d (need %d)", page_size, PAGE);
  JB_REFUSE(nkv <= 0 || nh % nkv != 0, "attention_prefix: %d heads are not a multiple of %d kv heads", nh, nkv);
  JB_REFUSE(hd <= 0 || hd > 256, "attention_prefix: head size %d", hd);
  const Step s{t.prefix_pages, t.block_table, t.q_start, t.kv_len, t.positions, prefix_len, z.ld_table, z.width, T, n_seqs, nh, nkv, hd, z.scale * LOG2E};
  const float *qf = (const float*)q, *kf = (const float*)k_cache, *vf = (const float*)v_cache;
  float* of = (float*)out;
  float* part_o = scratch;
  float2* ml = (float2*)(scratch + (size_t)(splits + own_slots) * T * nh * hd);
  if (hd % 4 != 0 || (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15)) {
    jb::Launch cfg(dim3((unsigned)(((long long)T * nh + 3) / 4)), dim3(128), 0, stream);
    return (int)cudaLaunchKernelEx(&cfg.c, rows_f32_kernel, qf, kf, vf, of, s);
  }
  JB_REFUSE((rows != 16 && rows != 64) || (own_rows != 16 && own_rows != 64) || own_slots < 1 || own_slots > 64 || splits < 0 ||
                splits > 64 || (splits > 0 && prefix_len <= 0) || (splits == 0 && prefix_len > 0),
            "attention_prefix: %d ranges of a prefix of %d tokens, blocks of %d and %d rows", splits, prefix_len, rows, own_rows);
  const int G = nh / nkv;
  const Slots parts{splits, splits, 0, 1, 1};
  cudaError_t e = cudaSuccess;
  if (splits > 0)
    e = pick<false>(hd, rows, dim3(nkv, (unsigned)(((long long)T * G + rows - 1) / rows), splits), stream, qf, kf, vf, part_o, ml, s, parts,
                    own_slots, 0);
  if (e != cudaSuccess) return (int)e;
  const int row_blocks = (max_q_len * G + own_rows - 1) / own_rows;
  e = pick<true>(hd, own_rows, dim3(n_seqs, nkv * row_blocks, own_slots), stream, qf, kf, vf, part_o, ml, s, parts, own_slots, row_blocks);
  if (e == cudaSuccess) e = join_go<float>(stream, qf, kf, vf, of, part_o, ml, nullptr, s, parts, own_slots);
  return (int)e;
}
