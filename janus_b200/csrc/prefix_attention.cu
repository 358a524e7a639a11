// Attention of a step whose sequences share a prefix: every query sees the prefix's keys and its own sequence's, up to its
// own position.  Key i of the prefix lies in page prefix_pages[i / 64], key prefix_len + i of sequence b in page
// block_table[b][i / 64].  softmax(q K^T scale) V over both together; kv head of query head h is floor(h nkv / nh).
//
// A softmax over a union of key sets joins from the sets' (maximum m, sum l, weighted values O):
//   m = max m_i,  l = sum 2^(m_i - m) l_i,  O = sum 2^(m_i - m) O_i   (scores in units of log2).
// So the prefix is attended once for all: the rows of ALL sequences' tokens make tiles of 128 for the tensor cores, which walk
// the prefix's keys in ranges (`prefix_tc_kernel<SPLIT>`), while `own_kernel` walks each sequence's own pages; partial results
// are float32.  Steps whose sequences bring many tokens fill tiles by themselves: there a tile walks the prefix and then its own
// pages and nothing is joined (`prefix_tc_kernel<WHOLE>`).
#include <cuda.h>

#include "prefix_attention.cuh"
#include "tc_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// bfloat16: tiles of 128 (token, query head of one kv head) rows on the tcgen05 tensor cores.
//   warp 0     TMA producer: the Q tiles, then blocks of KB keys and values (128-byte swizzle), each in a ring of two
//   warp 1     one lane issues the products: S = Q K^T into tensor memory, O += P V with P from tensor memory
//   warps 2..  one thread a row: softmax in float32 against a reference maximum that is raised (and O rescaled) only when a
//              row's maximum has grown by 2^8; P, in bfloat16 as the tensor core takes it, over the first half of S
// Two tiles a CTA take turns on the tensor core (NT = 2); a single tile has two S buffers and works a block ahead.
// SPLIT: the rows are the step's tokens whatever sequence they belong to, the keys a range of the prefix's blocks; what is
// written is the partial result.  WHOLE: the rows are one sequence's, the keys all that they see.
// ---------------------------------------------------------------------------
constexpr int BM = 128;
constexpr float RESCALE_LOG2 = 8.0f;

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// A operand from tensor memory (lane = row, a 32-bit column = two consecutive bfloat16 of K)
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 2^x by the special-function unit (2 ulp); arguments are <= 8, -inf gives 0
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// MN-major operand (values: a 128-byte row holds 64 consecutive numbers of one key, 8 keys a 1,024-byte atom): the leading
// offset is the distance of the next 64 numbers, the stride offset that of the next 8 keys.
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr, uint32_t lead, uint32_t stride) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)((lead >> 4) & 0x3FFF) << 16 | (uint64_t)((stride >> 4) & 0x3FFF) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <int N>
__device__ __forceinline__ float row_max(const uint32_t* sr) {
  float m[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) m[e] = fmaxf(__uint_as_float(sr[e]), __uint_as_float(sr[N - 4 + e]));
#pragma unroll
  for (int c = 4; c + 8 <= N - 4; c += 8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = max3(m[e], __uint_as_float(sr[c + 2 * e]), __uint_as_float(sr[c + 2 * e + 1]));
  }
  return max3(m[0], m[1], fmaxf(m[2], m[3]));
}
// p[c] = 2^(s[c] scale + neg_ref) for N scores in sr; bfloat16 pairs over the first N / 2 words; returns their float32 sum.
template <int N>
__device__ __forceinline__ float exp_pack_sum(uint32_t* sr, float scale_log2, float neg_ref) {
  const jb::Pair s2 = jb::pair(scale_log2, scale_log2), n2 = jb::pair(neg_ref, neg_ref), one = jb::pair(1.0f, 1.0f);
  jb::Pair acc[4] = {0ull, 0ull, 0ull, 0ull};   // the bit pattern of (0.0f, 0.0f)
#pragma unroll
  for (int c = 0; c < N / 2; ++c) {
    const jb::Pair x = jb::fma2(jb::pair(__uint_as_float(sr[2 * c]), __uint_as_float(sr[2 * c + 1])), s2, n2);
    const float p0 = fast_exp2(jb::lo(x)), p1 = fast_exp2(jb::hi(x));
    acc[c & 3] = jb::fma2(jb::pair(p0, p1), one, acc[c & 3]);
    sr[c] = pack_bf16(p0, p1);
  }
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) sum += jb::lo(acc[e]) + jb::hi(acc[e]);
  return sum;
}

template <int HDC, int NT, int KB>
struct Tc {
  static constexpr int SLABS = HDC / 64;                       // 64-number slabs of a row
  static constexpr int Q_BYTES = SLABS * BM * 128, KV_BYTES = SLABS * KB * 128;
  static constexpr int BARS = 1 + 8 + 2 * 2 + 2 * NT;          // q_full; k, v full and empty x 2; s_full, p_full x 2; o_full, o_done
  static constexpr int SMEM = NT * Q_BYTES + 4 * KV_BYTES + BARS * 8 + 16 + 1024;
  static constexpr int THREADS = 64 + NT * 128;
  static constexpr int COLS = 2 * KB + NT * HDC <= 256 ? 256 : 512;
  static_assert(2 * KB + NT * HDC <= 512 && SMEM <= 232448, "tensor and shared memory of one CTA");
};

enum Form { SPLIT, WHOLE };

// part_o: [slot][token][head][hd] float32, not normalised; part_ml: [slot][token][head] (maximum in log2 units, sum)
template <int HDC, int NT, int KB, Form FORM>
__global__ void __launch_bounds__(Tc<HDC, NT, KB>::THREADS, 1) prefix_tc_kernel(
    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
    const bf16* __restrict__ q, const bf16* __restrict__ k_cache, const bf16* __restrict__ v_cache, bf16* __restrict__ out,
    float* __restrict__ part_o, float2* __restrict__ part_ml, const Step s, int n_splits, int* __restrict__ status) {
  typedef Tc<HDC, NT, KB> C;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t q_s = jb::smem_u32(smem), k_s = q_s + NT * C::Q_BYTES, v_s = k_s + 2 * C::KV_BYTES;
  uint64_t* bars = (uint64_t*)(smem + NT * C::Q_BYTES + 4 * C::KV_BYTES);
  uint32_t* tmem_slot = (uint32_t*)(bars + C::BARS);
  const uint32_t bar0 = jb::smem_u32(bars);
  const uint32_t q_full = bar0, k_full = bar0 + 8, k_empty = bar0 + 24, v_full = bar0 + 40, v_empty = bar0 + 56;
  // an S buffer belongs to a tile (NT = 2), or to the even or odd blocks of the one tile
  auto s_full = [&](int b) { return bar0 + 72 + 16 * b; };
  auto p_full = [&](int b) { return bar0 + 80 + 16 * b; };
  auto o_full = [&](int w) { return bar0 + 104 + 16 * w; };
  auto o_done = [&](int w) { return bar0 + 112 + 16 * w; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    jb::mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      jb::mbar_init(k_full + 8 * i, 1);
      jb::mbar_init(k_empty + 8 * i, 1);
      jb::mbar_init(v_full + 8 * i, 1);
      jb::mbar_init(v_empty + 8 * i, 1);
      jb::mbar_init(s_full(i), 1);
      jb::mbar_init(p_full(i), 128);
    }
    for (int w = 0; w < NT; ++w) {
      jb::mbar_init(o_full(w), 1);
      jb::mbar_init(o_done(w), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) jb::tmem_alloc<C::COLS>(jb::smem_u32(tmem_slot));
  jb::tc_fence_before();
  __syncthreads();
  jb::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  jb::pdl_wait();
  // (after the wait: a kernel that starts early may read what the launch before this one wrote)
  jb::pdl_launch_dependents();

  // ---- which rows, which keys ----
  const int G = s.nh / s.nkv, tpt = BM / G, kvh = blockIdx.x;
  int tok0, n_tok, seq = 0, first_pos = 0;                     // first token, tokens of all tiles
  int block0 = 0, n_shared, n_own = 0;                         // first block of the prefix, its blocks, own blocks
  const int total = min(s.T, max(s.q_start[s.n_seqs], 0));
  if constexpr (FORM == SPLIT) {
    tok0 = blockIdx.y * NT * tpt;
    n_tok = min(NT * tpt, total - tok0);
    const int blocks = (s.prefix_len + KB - 1) / KB;
    block0 = (int)((long long)blockIdx.z * blocks / n_splits);
    n_shared = (int)((long long)(blockIdx.z + 1) * blocks / n_splits) - block0;
  } else {
    seq = blockIdx.z;
    const int start = s.q_start[seq], q_len = s.q_start[seq + 1] - start, tile = gridDim.y - 1 - blockIdx.y;
    tok0 = start + tile * NT * tpt;
    n_tok = min(NT * tpt, q_len - tile * NT * tpt);
    first_pos = s.kv_len[seq] - q_len + tile * NT * tpt;
    const int see = first_pos + n_tok;                         // keys that the last token sees
    n_shared = (min(see, s.prefix_len) + KB - 1) / KB;
    n_own = (min(max(see - s.prefix_len, 0), s.width * PAGE) + KB - 1) / KB;
  }
  const int nb = n_tok > 0 ? n_shared + n_own : 0;
  const int nslab = (s.hd + 63) / 64;

  if (nb > 0 && warp == 0) {
    if (lane == 0) {
      jb::mbar_expect_tx(q_full, NT * nslab * tpt * G * 128);   // a box holds tpt tokens x G heads
      for (int w = 0; w < NT; ++w)
        for (int h = 0; h < nslab; ++h) tma_load_4d(q_s + w * C::Q_BYTES + h * BM * 128, &map_q, q_full, h * 64, 0, kvh, tok0 + w * tpt);
      const int last_shared = (s.prefix_len - 1) / PAGE;
      const int last_own = FORM == WHOLE ? min((first_pos + n_tok - s.prefix_len - 1) / PAGE, s.width - 1) : 0;
      for (int j = 0; j < nb; ++j) {
        const int st = j & 1;
        int row0[KB / PAGE];
#pragma unroll
        for (int half = 0; half < KB / PAGE; ++half) {   // a block's second page may lie behind the last: those keys are masked
          int page;
          if (j < n_shared) page = s.prefix_pages[min((block0 + j) * (KB / PAGE) + half, last_shared)];
          else page = s.table[(size_t)seq * s.ld_table + min((j - n_shared) * (KB / PAGE) + half, last_own)];
          row0[half] = (max(page, 0) * s.nkv + kvh) * PAGE;
        }
        if (j >= 2 && !jb::mbar_wait(k_empty + 8 * st, ((j >> 1) - 1) & 1, status, 41)) break;
        jb::mbar_expect_tx(k_full + 8 * st, nslab * KB * 128);
#pragma unroll
        for (int half = 0; half < KB / PAGE; ++half)
          for (int h = 0; h < nslab; ++h)
            jb::tma_load_2d(k_s + st * C::KV_BYTES + h * KB * 128 + half * PAGE * 128, &map_k, k_full + 8 * st, h * 64, row0[half]);
        if (j >= 2 && !jb::mbar_wait(v_empty + 8 * st, ((j >> 1) - 1) & 1, status, 41)) break;
        jb::mbar_expect_tx(v_full + 8 * st, nslab * KB * 128);
#pragma unroll
        for (int half = 0; half < KB / PAGE; ++half)
          for (int h = 0; h < nslab; ++h)
            jb::tma_load_2d(v_s + st * C::KV_BYTES + h * KB * 128 + half * PAGE * 128, &map_v, v_full + 8 * st, h * 64, row0[half]);
      }
    }
  } else if (nb > 0 && warp == 1) {
    if (lane == 0) {
      const uint32_t idesc_s = jb::instr_desc_bf16(KB);
      const uint32_t idesc_o = jb::instr_desc_bf16((s.hd + 15) & ~15) | (1u << 16);   // values: MN-major
      bool ok = jb::mbar_wait(q_full, 0, status, 42);
      auto issue_s = [&](int w, int j) -> bool {
        const int st = j & 1, b = NT == 2 ? w : j & 1;
        if (!jb::mbar_wait(k_full + 8 * st, (j >> 1) & 1, status, 42)) return false;
        jb::tc_fence_after();
#pragma unroll
        for (int h = 0; h < C::SLABS; ++h) {
          const uint64_t a = jb::smem_desc_sw128(q_s + w * C::Q_BYTES + h * BM * 128);
          const uint64_t k = jb::smem_desc_sw128(k_s + st * C::KV_BYTES + h * KB * 128);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            if (h * 64 + ks * 16 < s.hd) jb::umma_bf16(tmem + b * KB, a + 2 * ks, k + 2 * ks, idesc_s, (h | ks) ? 1u : 0u);
        }
        jb::umma_commit(s_full(b));
        if (w == NT - 1) jb::umma_commit(k_empty + 8 * st);
        return true;
      };
      for (int w = 0; w < NT && ok; ++w) ok = issue_s(w, 0);
      for (int j = 0; j < nb && ok; ++j) {
        const int st = j & 1;
        if (NT == 1 && j + 1 < nb) ok = issue_s(0, j + 1);
        for (int w = 0; w < NT && ok; ++w) {
          const int b = NT == 2 ? w : j & 1;
          ok = jb::mbar_wait(p_full(b), (NT == 2 ? j : j >> 1) & 1, status, 42);
          if (ok && w == 0) ok = jb::mbar_wait(v_full + 8 * st, (j >> 1) & 1, status, 42);
          if (!ok) break;
          jb::tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < KB / 16; ++ks)
            umma_ts(tmem + 2 * KB + w * HDC, tmem + b * KB + ks * 8, desc_mn_sw128(v_s + st * C::KV_BYTES + ks * 2048, KB * 128, 1024),
                    idesc_o, (j | ks) ? 1u : 0u);
          jb::umma_commit(o_full(w));
          if (j == nb - 1) jb::umma_commit(o_done(w));
          if (w == NT - 1) jb::umma_commit(v_empty + 8 * st);
          if (NT == 2 && j + 1 < nb) ok = issue_s(w, j + 1);
        }
      }
    }
  } else if (n_tok > 0 && warp >= 2) {
    const int w = (warp - 2) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const int tl = w * tpt + row / G, token = tok0 + tl, head = kvh * G + row % G;
    const bool valid = row < tpt * G && tl < n_tok;
    int see_shared = 0, see_own = 0;                           // keys that the row sees
    if (valid) {
      const int see = (FORM == SPLIT ? s.positions[token] : first_pos + tl) + 1;
      see_shared = min(see, s.prefix_len);
      see_own = see - s.prefix_len;
    }
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16), o_col = 2 * KB + w * HDC;
    float m_ref = -CUDART_INF_F, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < nb && ok; ++j) {
      const int b = NT == 2 ? w : j & 1;
      ok = jb::mbar_wait(s_full(b), (NT == 2 ? j : j >> 1) & 1, status, 43);
      if (!ok) break;
      jb::tc_fence_after();
      uint32_t sr[KB];
#pragma unroll
      for (int c0 = 0; c0 < KB; c0 += 16) tmem_ld16(lane_addr + b * KB + c0, sr + c0);
      jb::tmem_ld_wait();
      const int see = j < n_shared ? see_shared - (block0 + j) * KB : see_own - (j - n_shared) * KB;
      if (see < KB) {
#pragma unroll
        for (int c = 0; c < KB; ++c)
          if (c >= see) sr[c] = 0xff800000u;   // -inf
      }
      const float mx = row_max<KB>(sr) * s.scale_log2;
      // loads and stores of tensor memory are warp-wide: a warp rescales together if any of its rows has to
      const bool grow = mx > m_ref + RESCALE_LOG2 || (m_ref == -CUDART_INF_F && mx > -CUDART_INF_F);
      if (__any_sync(0xffffffffu, grow)) {
        const float m_new = fmaxf(m_ref, mx);
        if (j > 0) {
          ok = jb::mbar_wait(o_full(w), (j - 1) & 1, status, 43);
          if (!ok) break;
          jb::tc_fence_after();
          const float corr = m_new == -CUDART_INF_F ? 1.0f : exp2f(m_ref - m_new);
#pragma unroll
          for (int c0 = 0; c0 < HDC; c0 += 16) {
            if (c0 >= s.hd) break;
            uint32_t r[16];
            tmem_ld16(lane_addr + o_col + c0, r);
            jb::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * corr);
            tmem_st16(lane_addr + o_col + c0, r);
          }
          tmem_st_wait();
          l *= corr;
        }
        m_ref = m_new;
      }
      l += exp_pack_sum<KB>(sr, s.scale_log2, m_ref == -CUDART_INF_F ? 0.0f : -m_ref);
#pragma unroll
      for (int c0 = 0; c0 < KB / 2; c0 += 16) tmem_st16(lane_addr + b * KB + c0, sr + c0);
      tmem_st_wait();
      jb::tc_fence_before();
      jb::mbar_arrive(p_full(b));
    }
    if (ok && nb > 0) ok = jb::mbar_wait(o_done(w), 0, status, 43);
    if (ok) {
      jb::tc_fence_after();
      const size_t place = (size_t)token * s.nh + head;
      if constexpr (FORM == SPLIT) {
        const size_t item = (size_t)blockIdx.z * s.T * s.nh + place;
        if (valid) part_ml[item] = make_float2(m_ref, l);
#pragma unroll
        for (int c0 = 0; c0 < HDC; c0 += 16) {
          if (c0 >= s.hd) break;
          uint32_t r[16];
          tmem_ld16(lane_addr + o_col + c0, r);   // warp-wide: rows without a token load too and store nothing
          jb::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            if (valid && c0 + i < s.hd)
              *reinterpret_cast<uint4*>(part_o + item * s.hd + c0 + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        }
      } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        bool finite = true;
#pragma unroll
        for (int c0 = 0; c0 < HDC; c0 += 16) {
          if (c0 >= s.hd) break;
          uint32_t r[16];
          if (nb > 0) {
            tmem_ld16(lane_addr + o_col + c0, r);
            jb::tmem_ld_wait();
          }
          uint32_t p[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = nb > 0 ? __uint_as_float(r[2 * i]) * inv : 0.0f, c = nb > 0 ? __uint_as_float(r[2 * i + 1]) * inv : 0.0f;
            finite = finite && (c0 + 2 * i >= s.hd || (isfinite(a) && isfinite(c)));
            p[i] = pack_bf16(a, c);
          }
          if (valid) {
            *reinterpret_cast<uint4*>(out + place * s.hd + c0) = make_uint4(p[0], p[1], p[2], p[3]);
            if (c0 + 8 < s.hd) *reinterpret_cast<uint4*>(out + place * s.hd + c0 + 8) = make_uint4(p[4], p[5], p[6], p[7]);
          }
        }
        unsigned again = __ballot_sync(0xffffffffu, valid && !finite);
        while (again) {
          const int l0 = __ffs(again) - 1;
          again &= again - 1;
          __syncwarp();
          one_row(q, k_cache, v_cache, out, s, seq, __shfl_sync(0xffffffffu, token, l0), __shfl_sync(0xffffffffu, head, l0));
        }
      }
    }
    jb::tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    jb::tc_fence_after();
    jb::tmem_dealloc<C::COLS>(tmem);
  }
}

// ---------------------------------------------------------------------------
// bfloat16: each sequence's own pages, by warp-level products.  A CTA has 16 (token, head) rows of one sequence and kv head and a
// range of its pages; each of its four warps takes 16 keys of every page through a ring of its own.
// ---------------------------------------------------------------------------
constexpr int OWN_THREADS = 128;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const bf16* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(jb::smem_u32(p)));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const bf16* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(jb::smem_u32(p)));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int HDC, int STAGES>
struct Own {
  static constexpr int LD = HDC + 8;                           // padded rows: an odd number of 16-byte pieces
  static constexpr int TILE = PAGE * LD, STAGE = 2 * TILE;
  static constexpr int RED_LD = HDC + 4;
  static constexpr int RED = (4 * 16 * RED_LD + 4 * 16 * 2) * 4;
  static constexpr int RING = STAGES * STAGE * 2;
  static constexpr int SMEM = 16 * LD * 2 + (RING > RED ? RING : RED);
};

// What is left to do with a row's sums over the warps: join them with the prefix's partial results and write the output
// (own_slots == 1), or leave them as one more partial result.
template <int HDC, int STAGES>
__global__ void __launch_bounds__(OWN_THREADS) own_kernel(const bf16* __restrict__ q, const bf16* __restrict__ k_cache,
                                                          const bf16* __restrict__ v_cache, bf16* __restrict__ out,
                                                          float* __restrict__ part_o, float2* __restrict__ part_ml, const Step s,
                                                          int prefix_slots, int own_slots, int row_blocks) {
  typedef Own<HDC, STAGES> C;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ int not_finite[16];
  bf16* q_s = reinterpret_cast<bf16*>(smem_raw);
  bf16* kv_s = q_s + 16 * C::LD;
  const int G = s.nh / s.nkv, seq = blockIdx.x, kvh = blockIdx.y / row_blocks, rb = blockIdx.y % row_blocks, split = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = s.hd;
  if (prefix_slots == 0) jb::pdl_wait();
  jb::pdl_launch_dependents();
  const int start = s.q_start[seq], q_len = s.q_start[seq + 1] - start;
  const int row0 = rb * 16, n_rows = min(16, q_len * G - row0);
  const int first_pos = s.kv_len[seq] - q_len;
  // own keys that the block's last row sees; pages are cut evenly among the splits
  const int see = n_rows > 0 ? first_pos + (row0 + n_rows - 1) / G + 1 - s.prefix_len : 0;
  const int pages = min(see > 0 ? (see + PAGE - 1) / PAGE : 0, s.width);
  const int p_begin = (int)((long long)split * pages / own_slots), p_end = (int)((long long)(split + 1) * pages / own_slots);
  const int* table = s.table + (size_t)seq * s.ld_table;
  uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  const int chunks = hd / 8;
  auto issue = [&](int p, int st) {
    const size_t row = ((size_t)max(table[p], 0) * s.nkv + kvh) * PAGE + warp * 16;
    const uint32_t k_d = jb::smem_u32(kv_s + (size_t)st * C::STAGE + warp * 16 * C::LD), v_d = k_d + C::TILE * 2;
    for (int ch = lane; ch < 16 * chunks; ch += 32) {
      const int r = ch / chunks, c = ch % chunks;
      cp_async16(k_d + (r * C::LD + c * 8) * 2, k_cache + (row + r) * hd + c * 8, policy);
      cp_async16(v_d + (r * C::LD + c * 8) * 2, v_cache + (row + r) * hd + c * 8, policy);
    }
  };
  if (p_begin < p_end) {
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      if (p_begin + i < p_end) issue(p_begin + i, i);
      cp_async_commit();
    }
    if (hd < HDC) {   // columns behind the head's numbers
      const int pad = HDC - hd;
      for (int i = threadIdx.x; i < STAGES * 2 * PAGE * pad; i += OWN_THREADS)
        kv_s[(size_t)(i / pad) * C::LD + hd + i % pad] = __float2bfloat16_rn(0.0f);
    }
    for (int i = threadIdx.x; i < 16 * (HDC / 8); i += OWN_THREADS) {
      const int r = i / (HDC / 8), c = i % (HDC / 8), rr = row0 + r;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (r < n_rows && c * 8 < hd)
        v = *reinterpret_cast<const uint4*>(q + ((size_t)(start + rr / G) * s.nh + kvh * G + rr % G) * hd + c * 8);
      *reinterpret_cast<uint4*>(q_s + r * C::LD + c * 8) = v;
    }
  }
  float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.0f, 0.0f}, o[HDC / 8][4];
#pragma unroll
  for (int j = 0; j < HDC / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
  int see_row[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = (lane >> 2) + 8 * r;
    see_row[r] = row < n_rows ? first_pos + (row0 + row) / G + 1 - s.prefix_len : 0;
  }
  __syncthreads();
  for (int p = p_begin; p < p_end; ++p) {
    const int st = (p - p_begin) % STAGES;
    if (p + STAGES - 1 < p_end) issue(p + STAGES - 1, (p - p_begin + STAGES - 1) % STAGES);
    cp_async_commit();
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const bf16* k_t = kv_s + (size_t)st * C::STAGE + warp * 16 * C::LD;
    const bf16* v_t = k_t + C::TILE;
    float x[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < HDC / 16; ++ks) {
      if (ks * 16 >= hd) break;
      uint32_t a[4], b[4];
      ldmatrix_x4(a, q_s + (lane & 15) * C::LD + ks * 16 + (lane >> 4) * 8);
      ldmatrix_x4(b, k_t + ((lane & 7) + ((lane >> 4) << 3)) * C::LD + ks * 16 + ((lane >> 3) & 1) * 8);
      mma_bf16(x[0], a, b[0], b[1]);
      mma_bf16(x[1], a, b[2], b[3]);
    }
    float mx[2] = {-CUDART_INF_F, -CUDART_INF_F}, corr[2], ref[2];
    const int key0 = p * PAGE + warp * 16 + 2 * (lane & 3);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[j][e] = key0 + j * 8 + (e & 1) < see_row[e >> 1] ? x[j][e] * s.scale_log2 : -CUDART_INF_F;
        mx[e >> 1] = fmaxf(mx[e >> 1], x[j][e]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      const float m_new = fmaxf(m[r], mx[r]);
      ref[r] = m_new == -CUDART_INF_F ? 0.0f : m_new;
      corr[r] = exp2f(m[r] - ref[r]);
      m[r] = m_new;
      l[r] *= corr[r];
    }
#pragma unroll
    for (int j = 0; j < HDC / 8; ++j) o[j][0] *= corr[0], o[j][1] *= corr[0], o[j][2] *= corr[1], o[j][3] *= corr[1];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[j][e] = exp2f(x[j][e] - ref[e >> 1]);
        l[e >> 1] += x[j][e];
      }
    uint32_t a[4] = {pack_bf16(x[0][0], x[0][1]), pack_bf16(x[0][2], x[0][3]), pack_bf16(x[1][0], x[1][1]), pack_bf16(x[1][2], x[1][3])};
#pragma unroll
    for (int j = 0; j < HDC / 8; j += 2) {
      if (j * 8 >= hd) break;
      uint32_t b[4];
      ldmatrix_x4_trans(b, v_t + (lane & 15) * C::LD + j * 8 + (lane >> 4) * 8);
      mma_bf16(o[j], a, b[0], b[1]);
      mma_bf16(o[j + 1], a, b[2], b[3]);
    }
    __syncwarp();
  }
  // ---- the warps' results meet in shared memory ----
  __syncthreads();
  float* red_o = reinterpret_cast<float*>(kv_s);
  float* red_ml = red_o + 4 * 16 * C::RED_LD;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = warp * 16 + (lane >> 2) + 8 * r;
    if ((lane & 3) == 0) {
      red_ml[2 * row] = m[r];
      red_ml[2 * row + 1] = l[r];
    }
#pragma unroll
    for (int j = 0; j < HDC / 8; ++j)
      *reinterpret_cast<float2*>(red_o + row * C::RED_LD + j * 8 + 2 * (lane & 3)) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
  }
  if (threadIdx.x < 16) not_finite[threadIdx.x] = 0;
  __syncthreads();
  if (prefix_slots > 0) jb::pdl_wait();   // the prefix's partial results are there
  finish_rows<bf16, 4, 16, OWN_THREADS>(q, k_cache, v_cache, out, part_o, part_ml, s, red_o, red_ml, C::RED_LD, not_finite, max(n_rows, 0),
                                        row0, start, seq, kvh, prefix_slots, own_slots, split);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
bool make_maps(CUtensorMap* mq, CUtensorMap* mk, CUtensorMap* mv, const void* q, const void* k, const void* v, const Step& s, int n_pages) {
  static jb::EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess)
      return false;
    fn = (jb::EncodeTiledFn)p;
  }
  const cuuint32_t el[4] = {1, 1, 1, 1};
  {
    const cuuint64_t G = s.nh / s.nkv, hd = s.hd;
    const cuuint64_t dims[4] = {hd, G, (cuuint64_t)s.nkv, (cuuint64_t)s.T}, strides[3] = {hd * 2, G * hd * 2, (cuuint64_t)s.nh * hd * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)G, 1, (cuuint32_t)(BM / G)};
    if (fn(mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(q), dims, strides, box, el, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  }
  for (int which = 0; which < 2; ++which) {
    const cuuint64_t dims[2] = {(cuuint64_t)s.hd, (cuuint64_t)n_pages * s.nkv * PAGE}, strides[1] = {(cuuint64_t)s.hd * 2};
    const cuuint32_t box[2] = {64, PAGE};
    if (fn(which ? mv : mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(which ? v : k), dims, strides, box, el,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  }
  return true;
}

template <int HDC, int NT, int KB, Form FORM>
cudaError_t tc_go(dim3 grid, cudaStream_t stream, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const bf16* q,
                  const bf16* k, const bf16* v, bf16* out, float* part_o, float2* part_ml, const Step& s, int splits, int* status) {
  typedef Tc<HDC, NT, KB> C;
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(prefix_tc_kernel<HDC, NT, KB, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    configured = true;
  }
  jb::Launch cfg(grid, dim3(C::THREADS), C::SMEM, stream);
  return cudaLaunchKernelEx(&cfg.c, prefix_tc_kernel<HDC, NT, KB, FORM>, mq, mk, mv, q, k, v, out, part_o, part_ml, s, splits, status);
}

template <int HDC, int STAGES>
cudaError_t own_go(dim3 grid, cudaStream_t stream, const bf16* q, const bf16* k, const bf16* v, bf16* out, float* part_o, float2* part_ml,
                   const Step& s, int prefix_slots, int own_slots, int row_blocks) {
  typedef Own<HDC, STAGES> C;
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(own_kernel<HDC, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    configured = true;
  }
  jb::Launch cfg(grid, dim3(OWN_THREADS), C::SMEM, stream);
  return cudaLaunchKernelEx(&cfg.c, own_kernel<HDC, STAGES>, q, k, v, out, part_o, part_ml, s, prefix_slots, own_slots, row_blocks);
}

}  // namespace

// bfloat16.  splits = 0: tiles of one sequence each walk all their keys (WHOLE).  Else the prefix's keys in `splits` ranges for all
// rows together and the own keys in `own_slots` ranges a sequence; part_o [splits (+ own_slots if > 1)][T][nh][hd] float32 and
// part_ml [..][T][nh][2] are scratch.  tiles: row tiles a CTA, 1 or 2.
JB_EXPORT int jb_attention_prefix_bf16(const void* q, const void* k_cache, const void* v_cache, void* out, float* part_o, float* part_ml,
                                       const int* prefix_pages, int prefix_len, const int* block_table, int ld_table, int width,
                                       const int* q_start, const int* kv_len, const int* positions, int T, int n_pages, int n_seqs,
                                       int nh, int nkv, int hd, int page_size, float scale, int max_q_len, int tiles, int splits,
                                       int own_slots, int* status, cudaStream_t stream) {
  if (T <= 0 || n_seqs <= 0 || max_q_len <= 0) return 0;
  JB_REFUSE(page_size != PAGE, "attention_prefix: page size %d (need %d)", page_size, PAGE);
  JB_REFUSE(nkv <= 0 || nh % nkv != 0, "attention_prefix: %d heads are not a multiple of %d kv heads", nh, nkv);
  JB_REFUSE(hd <= 0 || hd > 256 || hd % 8 != 0, "attention_prefix: bfloat16 heads of %d numbers (multiples of 8 up to 256)", hd);
  const int G = nh / nkv;
  JB_REFUSE(G > BM, "attention_prefix: %d query heads per kv head are more than %d", G, BM);
  JB_REFUSE(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15, "attention_prefix: operands must be 16-byte aligned");
  JB_REFUSE((long long)n_pages * nkv * PAGE > 0x7fffffffll, "attention_prefix: %d pages of %d heads are more rows than a tensor map counts",
            n_pages, nkv);
  JB_REFUSE(splits < 0 || own_slots < 1 || splits > (prefix_len + 127) / 128, "attention_prefix: %d ranges of a prefix of %d tokens", splits,
            prefix_len);
  const Step s{prefix_pages, block_table, q_start, kv_len, positions, prefix_len, ld_table, width, T, n_seqs, nh, nkv, hd, scale * LOG2E};
  const bf16 *qb = (const bf16*)q, *kb = (const bf16*)k_cache, *vb = (const bf16*)v_cache;
  bf16* ob = (bf16*)out;
  float2* ml = (float2*)part_ml;
  const bool whole = splits == 0 && prefix_len > 0;
  cudaError_t e = cudaSuccess;
  if (whole || splits > 0) {
    CUtensorMap mq, mk, mv;
    if (!make_maps(&mq, &mk, &mv, q, k_cache, v_cache, s, n_pages)) return JB_ERR_TENSORMAP;
    const int tpt = BM / G, nt = hd > 128 ? 1 : tiles;
    if (whole) {
      const dim3 grid(nkv, (max_q_len + nt * tpt - 1) / (nt * tpt), n_seqs);
      if (hd > 128) return (int)tc_go<256, 1, 64, WHOLE>(grid, stream, mq, mk, mv, qb, kb, vb, ob, nullptr, nullptr, s, 0, status);
      if (hd > 64)
        return (int)(nt == 2 ? tc_go<128, 2, 128, WHOLE>(grid, stream, mq, mk, mv, qb, kb, vb, ob, nullptr, nullptr, s, 0, status)
                             : tc_go<128, 1, 128, WHOLE>(grid, stream, mq, mk, mv, qb, kb, vb, ob, nullptr, nullptr, s, 0, status));
      return (int)(nt == 2 ? tc_go<64, 2, 128, WHOLE>(grid, stream, mq, mk, mv, qb, kb, vb, ob, nullptr, nullptr, s, 0, status)
                           : tc_go<64, 1, 128, WHOLE>(grid, stream, mq, mk, mv, qb, kb, vb, ob, nullptr, nullptr, s, 0, status));
    }
    const dim3 grid(nkv, (T + nt * tpt - 1) / (nt * tpt), splits);
    if (hd > 128) e = tc_go<256, 1, 64, SPLIT>(grid, stream, mq, mk, mv, qb, kb, vb, ob, part_o, ml, s, splits, status);
    else if (hd > 64)
      e = nt == 2 ? tc_go<128, 2, 128, SPLIT>(grid, stream, mq, mk, mv, qb, kb, vb, ob, part_o, ml, s, splits, status)
                  : tc_go<128, 1, 128, SPLIT>(grid, stream, mq, mk, mv, qb, kb, vb, ob, part_o, ml, s, splits, status);
    else
      e = nt == 2 ? tc_go<64, 2, 128, SPLIT>(grid, stream, mq, mk, mv, qb, kb, vb, ob, part_o, ml, s, splits, status)
                  : tc_go<64, 1, 128, SPLIT>(grid, stream, mq, mk, mv, qb, kb, vb, ob, part_o, ml, s, splits, status);
    if (e != cudaSuccess) return (int)e;
  }
  const int row_blocks = (max_q_len * G + 15) / 16;
  const dim3 grid(n_seqs, nkv * row_blocks, own_slots);
  if (hd > 128) e = own_go<256, 2>(grid, stream, qb, kb, vb, ob, part_o, ml, s, splits, own_slots, row_blocks);
  else if (hd > 64) e = own_go<128, 3>(grid, stream, qb, kb, vb, ob, part_o, ml, s, splits, own_slots, row_blocks);
  else e = own_go<64, 3>(grid, stream, qb, kb, vb, ob, part_o, ml, s, splits, own_slots, row_blocks);
  if (e != cudaSuccess) return (int)e;
  if (own_slots > 1) {
    jb::Launch cfg(dim3((unsigned)(((long long)T * nh + 3) / 4)), dim3(128), 0, stream);
    e = cudaLaunchKernelEx(&cfg.c, join_kernel<bf16>, qb, kb, vb, ob, (const float*)part_o, (const float2*)ml, s, splits + own_slots);
  }
  return (int)e;
}
