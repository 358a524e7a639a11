// Attention of beams over a paged cache, one query token a beam, compiled for one head size (-DJB_HEAD_DIM=..., a multiple of 8 up to
// 256; in shared memory rows are zero-padded to the next multiple of 16, the k extent of one MMA).
//
//   out_i = softmax(q_i K_i' scale) V_i over the first kv_len[i] keys of beam i; scores, maximum and sum in float32, weights
//   rounded to bfloat16 for the product with V, whose accumulators are float32.
//
// Beams of a request hold the same pages up to where they parted.  The rows of a tile are the (beam, query head) pairs of one key
// head, so that a shared page is read once for all beams; behind it every beam's own pages follow, one beam after another, for
// the rows of that beam alone.  A softmax over a union of keys joins from (maximum, sum, weighted values), whoever made the parts.
#include <math_constants.h>
#include <stdio.h>

#include "common.cuh"

#ifndef JB_HEAD_DIM
#define JB_HEAD_DIM 128
#endif

namespace {

typedef __nv_bfloat16 bf16;

constexpr int HD = JB_HEAD_DIM;
static_assert(HD % 8 == 0 && HD >= 8 && HD <= 256, "head size must be a multiple of 8 in [8, 256]");
constexpr int HDP = (HD + 15) / 16 * 16;
constexpr int PAGE = 64;
constexpr int LD = HDP + 8;                        // padded row: an odd number of 16-byte chunks, conflict-free ldmatrix
constexpr int CHUNKS = HD / 8;
constexpr int THREADS = 128;
constexpr int TILE = PAGE * LD, STAGE = 2 * TILE;  // elements
constexpr int STAGES = HD > 128 ? 2 : 3;
constexpr int MT = HD > 128 ? 1 : 2;               // row tiles of 16 a block: what the registers hold of float32 results
constexpr int ROWS = 16 * MT;
constexpr int RED_LD = HD + 8;
constexpr int MOST_BEAMS = 32;
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  const bf16* q;
  const bf16* k_cache;
  const bf16* v_cache;
  bf16* out;
  float* part_o;       // [rows of beams][heads][splits][HD], not divided by their sums
  float* part_ml;      // ... [2]: maximum (in units of log2), sum
  const int* table;
  const int* kv_len;
  const int* shared;
  int R, K, nh, nkv, W, n_pages, splits;
  float scale_log2;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// What a block reads next: a page, how many of its keys count, and for whose rows (-1: all that share it).
struct Unit {
  int page, keys, beam;
};

__global__ void __launch_bounds__(THREADS) beam_attention_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  bf16* q_s = reinterpret_cast<bf16*>(smem_raw);       // [ROWS][LD]
  bf16* kv_s = q_s + ROWS * LD;                        // [STAGES][K [64][LD], V [64][LD]]; the warps' exchange at the end
  __shared__ int length_s[MOST_BEAMS], first_s[MOST_BEAMS];   // keys of a beam; its first page of its own
  __shared__ int upto_s[MOST_BEAMS];                   // own pages of the beams up to this one
  __shared__ int shared_s, head_s;
  jb::pdl_launch_dependents();
  const int K = a.K, G = a.nh / a.nkv, blocks = (K * G + ROWS - 1) / ROWS;
  const int split = blockIdx.x, kvh = blockIdx.y / blocks, rho0 = blockIdx.y % blocks * ROWS, r = blockIdx.z;
  const int n_rows = min(ROWS, K * G - rho0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  jb::pdl_wait();
  // ---- which pages: shared ones first, then each beam's own (of the beams whose rows the block has) ----
  const int beam0 = rho0 / G, beam1 = (rho0 + n_rows - 1) / G;
  if (warp == 0) {
    const int len = lane < K ? min(max(a.kv_len[r * K + lane], 0), a.W * PAGE) : 0, pages = (len + PAGE - 1) / PAGE;
    const int most = __reduce_max_sync(0xffffffffu, len);
    const int head = __ffs(__ballot_sync(0xffffffffu, lane < K && len == most)) - 1;
    const int common = min(max(a.shared[r], 0), most / PAGE);
    const int first = len < common * PAGE ? 0 : common;      // shorter beams read all they have by themselves
    int n = lane >= beam0 && lane <= beam1 ? pages - first : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += t;
    }
    length_s[lane] = len;
    first_s[lane] = first;
    upto_s[lane] = n;
    if (lane == 0) shared_s = common, head_s = head;
  }
  __syncthreads();
  const int common = shared_s, units = common + upto_s[beam1];
  const int* head_pages = a.table + ((size_t)r * K + head_s) * a.W;
  const int u_start = (int)((long long)split * units / a.splits), u_end = (int)((long long)(split + 1) * units / a.splits);
  auto unit_of = [&](int u) {
    Unit x;
    if (u < common) {
      x.page = head_pages[u];
      x.keys = PAGE;
      x.beam = -1;
    } else {
      const int i = u - common;
      int b = beam0;
      while (upto_s[b] <= i) ++b;
      const int column = first_s[b] + i - (b > 0 ? upto_s[b - 1] : 0);
      x.page = a.table[((size_t)r * K + b) * a.W + column];
      x.keys = min(PAGE, length_s[b] - column * PAGE);
      x.beam = b;
    }
    if (x.page < 0 || x.page >= a.n_pages) x.page = 0, x.keys = 0;     // no page: no keys
    return x;
  };
  // Every warp loads, waits for and computes its own 16 keys of each page: no barrier of the block in the loop.
  auto issue = [&](const Unit& x, int stage) {
    const size_t row0 = ((size_t)x.page * a.nkv + kvh) * PAGE + warp * 16;
    bf16* k_rows = kv_s + (size_t)stage * STAGE + warp * 16 * LD;
    bf16* v_rows = k_rows + TILE;
    for (int ch = lane; ch < 16 * CHUNKS; ch += 32) {
      const int row = ch / CHUNKS, col = ch % CHUNKS;
      cp_async16(k_rows + row * LD + col * 8, a.k_cache + (row0 + row) * HD + col * 8);
      cp_async16(v_rows + row * LD + col * 8, a.v_cache + (row0 + row) * HD + col * 8);
    }
  };
  if constexpr (HDP != HD) {         // columns behind the head's numbers are never loaded
    constexpr int PAD = HDP > HD ? HDP - HD : 1;
    for (int i = threadIdx.x; i < STAGES * 2 * PAGE * PAD; i += THREADS) kv_s[(i / PAD) * LD + HD + i % PAD] = __float2bfloat16_rn(0.0f);
  }
  Unit ring[STAGES];
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (u_start + s < u_end) {
      ring[s] = unit_of(u_start + s);
      issue(ring[s], s);
    }
    cp_async_commit();
  }
  for (int ch = threadIdx.x; ch < ROWS * (HDP / 8); ch += THREADS) {
    const int row = ch / (HDP / 8), col = ch % (HDP / 8), rho = rho0 + row;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (row < n_rows && col < CHUNKS)
      v = *reinterpret_cast<const uint4*>(a.q + (((size_t)r * K + rho / G) * a.nh + kvh * G + rho % G) * HD + col * 8);
    *reinterpret_cast<uint4*>(q_s + row * LD + col * 8) = v;
  }
  __syncthreads();
  int beam_of[MT][2];                // of this thread's rows; -1: no row
  bool joins[MT][2];                 // whether the row reads the shared pages
  float m[MT][2], l[MT][2], o[MT][HDP / 8][4];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = t * 16 + (lane >> 2) + 8 * h;
      beam_of[t][h] = row < n_rows ? (rho0 + row) / G : -1;
      joins[t][h] = row < n_rows && length_s[beam_of[t][h]] >= common * PAGE;
      m[t][h] = -CUDART_INF_F;
      l[t][h] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < HDP / 8; ++j) o[t][j][0] = o[t][j][1] = o[t][j][2] = o[t][j][3] = 0.0f;
  }
  const int c = lane & 3;
  for (int u0 = u_start; u0 < u_end; u0 += STAGES) {
#pragma unroll
    for (int stage = 0; stage < STAGES; ++stage) {
      const int u = u0 + stage;
      if (u >= u_end) break;
      constexpr int AHEAD = STAGES - 1;
      if (u + AHEAD < u_end) {
        ring[(stage + AHEAD) % STAGES] = unit_of(u + AHEAD);
        issue(ring[(stage + AHEAD) % STAGES], (stage + AHEAD) % STAGES);
      }
      cp_async_commit();
      cp_async_wait<AHEAD>();
      __syncwarp();
      const Unit x = ring[stage];
      bf16* k_tile = kv_s + (size_t)stage * STAGE + warp * 16 * LD;
      bf16* v_tile = k_tile + TILE;
      const int keys = x.keys - warp * 16;            // of this warp's 16
      if (keys > 0) {
        if (keys < 16) {                              // values behind the last key: a weight of 0 does not silence what is no number
          for (int i = lane; i < (16 - keys) * (HDP / 8); i += 32)
            *reinterpret_cast<uint4*>(v_tile + (keys + i / (HDP / 8)) * LD + i % (HDP / 8) * 8) = make_uint4(0u, 0u, 0u, 0u);
          __syncwarp();
        }
        bool skip[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t)
          skip[t] = x.beam >= 0 && ((x.beam + 1) * G <= rho0 + t * 16 || x.beam * G >= rho0 + t * 16 + 16);
        float s[MT][2][4];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int j = 0; j < 2; ++j) s[t][j][0] = s[t][j][1] = s[t][j][2] = s[t][j][3] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < HDP / 16; ++ks) {
          uint32_t b[4];
          ldmatrix_x4(b, k_tile + ((lane & 7) + ((lane >> 4) << 3)) * LD + ks * 16 + ((lane >> 3) & 1) * 8);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            if (!skip[t]) {
              uint32_t qa[4];
              ldmatrix_x4(qa, q_s + (t * 16 + (lane & 15)) * LD + ks * 16 + (lane >> 4) * 8);
              mma_bf16(s[t][0], qa, b[0], b[1]);
              mma_bf16(s[t][1], qa, b[2], b[3]);
            }
          }
        }
        uint32_t pa[MT][4];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if (skip[t]) continue;
          float mx[2] = {-CUDART_INF_F, -CUDART_INF_F}, corr[2], use[2];
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int h = e >> 1, key = j * 8 + 2 * c + (e & 1);
              const bool ok = key < keys && (x.beam < 0 ? joins[t][h] : beam_of[t][h] == x.beam);
              s[t][j][e] = ok ? s[t][j][e] * a.scale_log2 : -CUDART_INF_F;
              mx[h] = fmaxf(mx[h], s[t][j][e]);
            }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            const float next = fmaxf(m[t][h], mx[h]);
            use[h] = next == -CUDART_INF_F ? 0.0f : next;
            corr[h] = exp2f(m[t][h] - use[h]);
            m[t][h] = next;
            l[t][h] *= corr[h];
          }
#pragma unroll
          for (int j = 0; j < HDP / 8; ++j) {
            o[t][j][0] *= corr[0];
            o[t][j][1] *= corr[0];
            o[t][j][2] *= corr[1];
            o[t][j][3] *= corr[1];
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[t][j][e] = exp2f(s[t][j][e] - use[e >> 1]);
              l[t][e >> 1] += s[t][j][e];
            }
          pa[t][0] = pack_bf16(s[t][0][0], s[t][0][1]);
          pa[t][1] = pack_bf16(s[t][0][2], s[t][0][3]);
          pa[t][2] = pack_bf16(s[t][1][0], s[t][1][1]);
          pa[t][3] = pack_bf16(s[t][1][2], s[t][1][3]);
        }
#pragma unroll
        for (int j = 0; j < HDP / 8; j += 2) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, v_tile + (lane & 15) * LD + j * 8 + (lane >> 4) * 8);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            if (!skip[t]) {
              mma_bf16(o[t][j], pa[t], b[0], b[1]);
              mma_bf16(o[t][j + 1], pa[t], b[2], b[3]);
            }
          }
        }
      }
      __syncwarp();   // the warp is done with its rows of this stage before its next loads overwrite them
    }
  }
  cp_async_wait<0>();
  __syncthreads();    // every warp has left the ring: its memory becomes the exchange
  float* red_o = reinterpret_cast<float*>(kv_s);             // [4][ROWS][RED_LD]
  float* red_ml = red_o + 4 * ROWS * RED_LD;                 // [4][ROWS][2]
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float sum = l[t][h];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const int row = t * 16 + (lane >> 2) + 8 * h;
      if (c == 0) red_ml[(warp * ROWS + row) * 2] = m[t][h], red_ml[(warp * ROWS + row) * 2 + 1] = sum;
#pragma unroll
      for (int j = 0; j < HDP / 8; ++j)
        if (j * 8 < HD)
          *reinterpret_cast<float2*>(red_o + (size_t)(warp * ROWS + row) * RED_LD + j * 8 + 2 * c) = make_float2(o[t][j][2 * h], o[t][j][2 * h + 1]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_rows * HD; i += THREADS) {
    const int row = i / HD, d = i % HD, rho = rho0 + row;
    float most = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < 4; ++w) most = fmaxf(most, red_ml[(w * ROWS + row) * 2]);
    const float use = most == -CUDART_INF_F ? 0.0f : most;
    float value = 0.0f, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2f(red_ml[(w * ROWS + row) * 2] - use);
      value += red_o[(size_t)(w * ROWS + row) * RED_LD + d] * f;
      sum += red_ml[(w * ROWS + row) * 2 + 1] * f;
    }
    const size_t item = ((size_t)r * K + rho / G) * a.nh + kvh * G + rho % G;
    if (a.splits == 1) {
      a.out[item * HD + d] = __float2bfloat16_rn(sum > 0.0f ? value / sum : 0.0f);
    } else {
      const size_t part = item * a.splits + split;
      if (most > -CUDART_INF_F) a.part_o[part * HD + d] = value;       // (a part without keys weighs nothing and is not read)
      if (d == 0) a.part_ml[part * 2] = most, a.part_ml[part * 2 + 1] = sum;
    }
  }
}

// A warp a (beam, head): the parts of its keys joined.
__global__ void __launch_bounds__(128) beam_attention_join_kernel(const Args a) {
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= (long long)a.R * a.K * a.nh) return;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + item * a.splits;
  float most = -CUDART_INF_F;
  for (int s = lane; s < a.splits; s += 32) most = fmaxf(most, ml[s].x);
  most = jb::warp_max(most);
  const float use = most == -CUDART_INF_F ? 0.0f : most;
  constexpr int N = (HD + 31) / 32;
  float o[N], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.0f;
  for (int s = 0; s < a.splits; ++s) {
    const float2 x = ml[s];
    if (x.x == -CUDART_INF_F) continue;
    const float f = exp2f(x.x - use);
    sum += x.y * f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * 32 + lane < HD) o[i] += a.part_o[(item * a.splits + s) * HD + i * 32 + lane] * f;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i * 32 + lane < HD) a.out[item * HD + i * 32 + lane] = __float2bfloat16_rn(sum > 0.0f ? o[i] / sum : 0.0f);
}

constexpr int RING_BYTES = STAGES * STAGE * 2, RED_BYTES = 4 * ROWS * (RED_LD + 2) * 4;
constexpr int SMEM = ROWS * LD * 2 + (RING_BYTES > RED_BYTES ? RING_BYTES : RED_BYTES);
static_assert(SMEM <= 227 * 1024, "shared memory of a block");

}  // namespace

// part: float32 scratch of R K nh splits (HD + 2) numbers where splits > 1.
JB_EXPORT int jb_attention_beams(const void* q, const void* k_cache, const void* v_cache, void* out, void* part, const int* table,
                                 const int* kv_len, const int* shared, int R, int K, int nh, int nkv, int W, int n_pages, int splits,
                                 float scale, cudaStream_t stream) {
  const int blocks = nkv > 0 && nh > 0 ? nkv * ((K * (nh / nkv) + ROWS - 1) / ROWS) : 0;
  JB_REFUSE(R < 1 || R > 65535 || K < 1 || K > MOST_BEAMS || nkv < 1 || nh < nkv || nh % nkv || W < 1 || W > 0x7fffffff / PAGE || n_pages < 1 ||
                splits < 1 || blocks > 65535,
            "attention_beams: %d groups of %d beams, %d heads over %d, %d pages a row, %d splits", R, K, nh, nkv, W, splits);
  static bool ready[64] = {};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return (int)e;
  if (device >= 64 || !ready[device]) {
    e = cudaFuncSetAttribute(beam_attention_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return (int)e;
    if (device < 64) ready[device] = true;
  }
  float* part_o = (float*)part;
  Args a{(const bf16*)q, (const bf16*)k_cache, (const bf16*)v_cache, (bf16*)out, part_o,
         part_o + (splits > 1 ? (size_t)R * K * nh * splits * HD : 0), table, kv_len, shared, R, K, nh, nkv, W, n_pages, splits, scale * LOG2E};
  jb::Launch cfg(dim3(splits, blocks, R), dim3(THREADS), SMEM, stream);
  e = cudaLaunchKernelEx(&cfg.c, beam_attention_kernel, a);
  if (e != cudaSuccess || splits == 1) return (int)e;
  jb::Launch join(dim3((unsigned)(((long long)R * K * nh + 3) / 4)), dim3(128), 0, stream);
  return (int)cudaLaunchKernelEx(&join.c, beam_attention_join_kernel, a);
}
