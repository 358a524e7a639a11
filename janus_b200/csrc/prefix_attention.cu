// Attention of a step whose sequences share a prefix: every query sees the prefix's keys and its own sequence's, up to its
// own position.  Key i of the prefix lies in page prefix_pages[i / 64], key prefix_len + i of sequence b in page
// block_table[b][i / 64].  softmax(q K^T scale) V over both together; kv head of query head h is floor(h nkv / nh).
//
// A softmax over a union of key sets joins from the sets' (maximum m, sum l, weighted values O):
//   m = max m_i,  l = sum 2^(m_i - m) l_i,  O = sum 2^(m_i - m) O_i   (scores in units of log2).
// So the prefix is attended once for all: the rows of ALL sequences' tokens make tiles of 128 for the tensor cores, which walk
// the prefix's keys in ranges (`prefix_tc_kernel<SHARED>`), and each sequence's own pages are walked (`own_kernel`; tiles again
// where a sequence brings many tokens, `<OWN>`); what they leave is float32 and is joined.  Where sequences bring many tokens behind a
// prefix that is not much longer, a tile walks the prefix and then its own pages and nothing is joined (`<WHOLE>`).  Few rows behind a
// short prefix walk it with their own keys (`own_kernel` alone): a launch less.
//
// The launches overlap (each begins before the one in front of it has ended, and asks for its results last).  What bounds them, of
// the measured 6,537 GB/s and 1,637 TFLOP/s, with 32 heads over 8 of 128 numbers:
//   64 single tokens behind 8,192, 30 to 700 own: 29 us; the prefix 18 us of them by 128 blocks, each waiting on its own row tile's
//     chain (scores, weights, values), the own keys' 40 MB beside it, 5 us for the join's launch and one round of loads
//   256 behind 16,384, 3 to 2,500 own: 122 us in the first 0.1 s of such calls, 140 once the power limit has lowered the clock; prefix
//     products at 1,100 TFLOP/s (of all multiprocessors) while they run, own keys at 5.2 TB/s while they do, each on a part of the
//     multiprocessors
//   8 prompts of up to 510 tokens behind 4,100: 99 us; the prefix 80 us at 57 % of the tensor pipe's cycles (a block of keys for two tiles
//     takes 3,400 cycles: 2,048 of products, 2,048 of the special-function unit, which hide each other in part), own keys the rest
#include <cuda.h>

#include "prefix_attention.cuh"
#include "tc_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// bfloat16: tiles of 128 (token, query head of one kv head) rows on the tcgen05 tensor cores.
//   warp 0     TMA producer: the Q tiles, then blocks of KB keys and values (128-byte swizzle), each in a ring of two
//   warp 1     one lane issues the products: S = Q K^T into tensor memory, O += P V with P from tensor memory
//   warps 2..  two threads a row, each with half of a block's keys: softmax in float32 against a reference maximum that is raised
//              (and O rescaled) only when a row's maximum has grown by 2^8; P, in bfloat16 as the tensor core takes it, over the
//              first half of S.  (With one thread a row the softmax took twice as long as the products it has to hide behind.)
// Two tiles a CTA take turns on the tensor core (NT = 2); a single tile has two S buffers and works a block ahead, or (SPLIT) is worked on
// by two groups, which work two blocks ahead and join their sums at the end.  P is handed over in
// two parts, 32 keys of each half first: their product with the values runs while the others' weights are made (8 prompts: 107 us
// with one, 103 with two).
// SHARED walks an even share of a list of (tile, kv head, key block), each share a partial result of every tile that it has a part of.
// A tile's places of the list may be more than its blocks, so that shares end where tiles do.
// ---------------------------------------------------------------------------
constexpr int BM = 128;
constexpr float RESCALE_LOG2 = 8.0f;

// Bounded wait: false (and *status = code) if the phase did not complete in 4e9 cycles, about two seconds.  The clock is read
// once in 64 tries, and it is the multiprocessor's own: the time in nanoseconds takes as long to read as a block's products.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, int* status, int code) {
  if (jb::mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (jb::mbar_try(bar, parity)) return true;
    if (clock64() - t0 > 4000000000ll) {
      atomicCAS(status, 0, code);
      return false;
    }
  }
}

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
// The same by multiply-adds: 2^f for |f| <= 1/2 by the cubic with value 1 at 0 and the least greatest relative error (1.0e-4, a
// twentieth of the rounding to bfloat16 that follows), the whole part added to the exponent's bits.  Anything to -127 gives 0 (a masked
// key's -inf must: a stale value may lie behind it), NaN a result that rounds to infinity, for which the row is made anew.
__device__ __forceinline__ float poly_exp2(float x) {
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(x), "f"(-127.0f));
  const float t = x + 12582912.0f;   // 1.5 x 2^23: the whole part in the low bits
  const float f = x - (t - 12582912.0f);
  const float p = fmaf(fmaf(fmaf(0.05500893f, f, 0.24221096f), f, 0.69328293f), f, 1.0f);
  return __int_as_float(__float_as_int(p) + (__float_as_int(t) << 23));
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
__device__ __forceinline__ jb::Pair add2(jb::Pair a, jb::Pair b) {
  jb::Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// p[c] = 2^(s[c] scale + neg_ref) for N scores in sr; bfloat16 pairs over the first N / 2 words; returns their float32 sum.
// POLY: one of eight by multiply-adds, while the special-function unit makes the others: with two tiles a block, each's weights are what
// the other's products wait for (8 prompts of up to 510 tokens behind 4,100: 104 and 100 us; one of four 103, and with more
// registers spill).  With one tile a block it changes nothing.
template <int N, bool POLY>
__device__ __forceinline__ float exp_pack_sum(uint32_t* sr, float scale_log2, float neg_ref) {
  const jb::Pair s2 = jb::pair(scale_log2, scale_log2), n2 = jb::pair(neg_ref, neg_ref);
  jb::Pair acc[4] = {0ull, 0ull, 0ull, 0ull};   // the bit pattern of (0.0f, 0.0f)
#pragma unroll
  for (int c = 0; c < N / 2; ++c) {
    const jb::Pair x = jb::fma2(jb::pair(__uint_as_float(sr[2 * c]), __uint_as_float(sr[2 * c + 1])), s2, n2);
    const bool poly = POLY && c % 8 == 7;
    const float p0 = poly ? poly_exp2(jb::lo(x)) : fast_exp2(jb::lo(x)), p1 = poly ? poly_exp2(jb::hi(x)) : fast_exp2(jb::hi(x));
    acc[c & 3] = add2(acc[c & 3], jb::pair(p0, p1));
    sr[c] = pack_bf16(p0, p1);
  }
  const jb::Pair all = add2(add2(acc[0], acc[1]), add2(acc[2], acc[3]));
  return jb::lo(all) + jb::hi(all);
}

template <int HDC, int NT, int KB>
struct Tc {
  static constexpr int SLABS = HDC / 64;                       // 64-number slabs of a row
  static constexpr int Q_BYTES = SLABS * BM * 128, KV_BYTES = SLABS * KB * 128;
  // Heads of up to 64 numbers, one tile: two groups of warps, each with every second block of 64 keys, sums and an O of its own, so that
  // one's weights are made while the other waits for scores (132 tokens behind 6,001: 28.9 -> 27.5 us, 100 behind 5,000 24.0 -> 22.3).
  // With 128 numbers it is between 9 % faster and 7 % slower: there the keys' way from L2 is what one tile's block waits for (64 KB for
  // 1.25 us of work, 6.7 TB/s of 128 blocks).
  static constexpr bool SPLIT = NT == 1 && HDC == 64;
  static constexpr int ST = SPLIT ? 4 : 2, SB = SPLIT ? 4 : 2, OB = SPLIT ? 2 : NT;   // stages of keys and of values; S and O buffers
  static constexpr int BARS = 1 + 4 * ST + 3 * SB + 3 * OB;    // q_full; k, v full and empty; s_full, p_half, p_full; o_full, o_done, o_free
  static constexpr int SWAP = NT * 2 * BM;                     // floats: what the two halves of a row tell each other
  static constexpr int SMEM = NT * Q_BYTES + 2 * ST * KV_BYTES + SWAP * 4 + NT * 4 * 4 + 8 + BARS * 8 + 16;
  static constexpr int THREADS = 64 + NT * 256;
  static constexpr int CHUNKS = KB / 64;                       // in which a block's weights are handed on
  // (one tile of up to 128 numbers a row: 96 registers a thread, as 576 threads have, so that a block of own_kernel finds registers
  // beside this one; rows of up to 64 leave enough anyway)
  static constexpr int BOUND = HDC == 128 ? 576 : THREADS;
  static constexpr int COLS = SB * KB + OB * HDC <= 256 ? 256 : 512;
  static_assert(SB * KB + OB * HDC <= 512 && SMEM <= 232448, "tensor and shared memory of one CTA");
};
// One lane of a warp whose lanes are all here.  (Work given to lane 0 by its number is not known to the compiler to be one thread's:
// every operand of a product then went through a vector register, and issuing products took twice as long as computing them.)
__device__ __forceinline__ bool elected() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0u;
}
// A barrier of two warps that tells both whether any of their threads says `yes`.
__device__ __forceinline__ bool pair_any(int barrier, bool yes) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)yes), "r"(barrier)
      : "memory");
  return any != 0u;
}
__device__ __forceinline__ void pair_sync(int barrier) { asm volatile("bar.sync %0, 64;" ::"r"(barrier) : "memory"); }

// SHARED: the step's tokens over the prefix, results left as parts.  WHOLE: one sequence's tokens over all that they see.  OWN: one
// sequence's tokens over its own keys, joined with the part over the prefix, or left as one more where there are several.
enum Form { SHARED, WHOLE, OWN };

__device__ __forceinline__ void store8(float* p, const uint32_t* r) {   // a whole 32-byte sector of a row
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
               "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void load8(const float* p, float* r) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
               : "l"(p)
               : "memory");
}

template <int HDC, int NT, int KB, Form FORM>
__global__ void __launch_bounds__(Tc<HDC, NT, KB>::BOUND, 1) prefix_tc_kernel(
    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
    const bf16* __restrict__ q, const bf16* __restrict__ k_cache, const bf16* __restrict__ v_cache, bf16* __restrict__ out,
    float* __restrict__ part_o, float2* __restrict__ part_ml, const Step s, const Slots parts, int* __restrict__ status) {
  typedef Tc<HDC, NT, KB> C;
  extern __shared__ __align__(1024) uint8_t smem[];            // (no static shared memory: it begins where it is declared to)
  const uint32_t q_s = jb::smem_u32(smem), k_s = q_s + NT * C::Q_BYTES, v_s = k_s + C::ST * C::KV_BYTES;
  float* swap = (float*)(smem + NT * C::Q_BYTES + 2 * C::ST * C::KV_BYTES);   // [tile][half][row]
  int* gave_up = (int*)(swap + C::SWAP);                       // [tile][quarter]: one of the two warps has
  int* found = gave_up + NT * 4;                               // WHOLE, OWN: the block's sequence and tile of it
  uint64_t* bars = (uint64_t*)(found + 2);
  uint32_t* tmem_slot = (uint32_t*)(bars + C::BARS);
  const uint32_t bar0 = jb::smem_u32(bars);
  const uint32_t q_full = bar0, k_full = bar0 + 8, k_empty = k_full + 8 * C::ST, v_full = k_empty + 8 * C::ST, v_empty = v_full + 8 * C::ST;
  const uint32_t s_bars = v_empty + 8 * C::ST, o_bars = s_bars + 24 * C::SB;
  // an S buffer belongs to a tile (NT = 2), to the even or odd blocks of the one tile, or (SPLIT) of one group's
  auto s_full = [&](int b) { return s_bars + 24 * b; };
  auto p_half = [&](int b) { return s_bars + 24 * b + 8; };
  auto p_full = [&](int b) { return s_bars + 24 * b + 16; };
  auto o_full = [&](int w) { return o_bars + 24 * w; };        // a block's product has landed in O
  auto o_done = [&](int w) { return o_bars + 24 * w + 8; };    // ... the last block's of a segment
  auto o_free = [&](int w) { return o_bars + 24 * w + 16; };   // O has been read and may be begun anew
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    jb::mbar_init(q_full, 1);
    for (int i = 0; i < C::ST; ++i) {
      jb::mbar_init(k_full + 8 * i, 1);
      jb::mbar_init(k_empty + 8 * i, 1);
      jb::mbar_init(v_full + 8 * i, 1);
      jb::mbar_init(v_empty + 8 * i, 1);
    }
    for (int i = 0; i < C::SB; ++i) {
      jb::mbar_init(s_full(i), 1);
      jb::mbar_init(p_half(i), 8);
      jb::mbar_init(p_full(i), C::SPLIT ? 4 : 8);   // an arrival a warp: one a thread would be 256 operations on one word
    }
    for (int w = 0; w < C::OB; ++w) {
      jb::mbar_init(o_full(w), 1);
      jb::mbar_init(o_done(w), 1);
      jb::mbar_init(o_free(w), 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < NT * 4) gave_up[threadIdx.x] = 0;
  if (warp == 1) jb::tmem_alloc<C::COLS>(jb::smem_u32(tmem_slot));
  jb::tc_fence_before();
  __syncthreads();
  jb::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  if (FORM != OWN || parts.most == 0) jb::pdl_wait();
  // WHOLE, OWN: which tile of which sequence this block has, by a list of the sequences' tiles (a grid of the longest one's would be
  // mostly blocks without work, and each has the multiprocessor to itself)
  if constexpr (FORM != SHARED) {
    if (warp == 2) {
      const int chunk = (s.n_seqs + 31) / 32, seq0 = min(lane * chunk, s.n_seqs), seq1 = min(seq0 + chunk, s.n_seqs), rows = NT * (BM / (s.nh / s.nkv));
      int mine = 0;
#pragma unroll 4
      for (int i = seq0; i < seq1; ++i) mine += (max(s.q_start[i + 1] - s.q_start[i], 0) + rows - 1) / rows;
      int up = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += t;
      }
      const int tile = blockIdx.y;
      if (lane == 0) found[0] = -1, found[1] = 0;
      __syncwarp();
      if (tile < up && tile >= up - mine) {
        int at = up - mine, i = seq0;
        for (;; ++i) {
          const int n = (max(s.q_start[i + 1] - s.q_start[i], 0) + rows - 1) / rows;
          if (tile < at + n) break;
          at += n;
        }
        found[0] = i, found[1] = (at + (max(s.q_start[i + 1] - s.q_start[i], 0) + rows - 1) / rows - 1) - tile;   // the longest first
      }
    }
    __syncthreads();
  }
  // (after the wait: a kernel that starts early may read what the launch before this one wrote)
  jb::pdl_launch_dependents();

  // ---- which rows, which keys: a list of segments, each one tile (or two) over a range of key blocks ----
  const int G = s.nh / s.nkv, tpt = BM / G;
  const int total_tokens = min(s.T, max(s.q_start[s.n_seqs], 0));
  struct Segment {
    int tok0, n_tok, kvh, block0, n_shared, nb;   // first token, tokens of all tiles; first block of the prefix, its blocks, all blocks
    int slot;
  };
  int seq = 0, seq_start = 0, seq_pos = 0;        // SHARED: not used
  const int flat_begin = FORM == SHARED ? blockIdx.x * parts.per : 0;
  const int flat_end = FORM == SHARED ? min(flat_begin + parts.per, (s.T + parts.tile_tokens - 1) / parts.tile_tokens * s.nkv * parts.blocks) : 1;
  if constexpr (FORM != SHARED) {
    seq = found[0];
    if (seq >= 0) seq_start = s.q_start[seq], seq_pos = s.kv_len[seq] - (s.q_start[seq + 1] - seq_start);
  }
  // the segment that begins at place `at` of the list; steps `at` on to the next
  auto segment = [&](int& at) {
    Segment g;
    if constexpr (FORM == SHARED) {
      const int item = at / parts.blocks;
      g.block0 = at - item * parts.blocks;
      g.nb = g.n_shared = min((s.prefix_len + KB - 1) / KB - g.block0, flat_end - at);
      g.kvh = item % s.nkv, g.tok0 = item / s.nkv * NT * tpt;
      g.n_tok = min(NT * tpt, total_tokens - g.tok0);
      g.slot = blockIdx.x - item * parts.blocks / parts.per;
      at += min(parts.blocks - g.block0, flat_end - at);
    } else {
      const int q_len = seq < 0 ? 0 : s.q_start[seq + 1] - seq_start, first = found[1] * NT * tpt;
      g.kvh = blockIdx.x, g.tok0 = seq_start + first, g.n_tok = min(NT * tpt, q_len - first), g.block0 = 0, g.slot = 0;
      const int see = seq_pos + first + g.n_tok;             // keys that the last token sees
      g.n_shared = FORM == WHOLE ? (max(min(see, s.prefix_len), 0) + KB - 1) / KB : 0;
      g.nb = g.n_tok > 0 ? g.n_shared + (min(max(see - s.prefix_len, 0), s.width * PAGE) + KB - 1) / KB : 0;
      ++at;
    }
    return g;
  };
  const int nslab = (s.hd + 63) / 64;

  if (warp == 0) {
    if (elected()) {
      const int last_shared = max((s.prefix_len - 1) / PAGE, 0);
      bool ok = true;
      int it = 0;                                             // blocks since the kernel's begin
      for (int at = flat_begin; at < flat_end && ok;) {
        const Segment g = segment(at);
        if (g.nb == 0) break;
        // every product with the queries before these is done when the last block's keys are free
        if (it > 0) ok = mbar_wait(k_empty + 8 * ((it - 1) % C::ST), (it - 1) / C::ST & 1, status, 41);
        if (!ok) break;
        jb::mbar_expect_tx(q_full, NT * nslab * tpt * G * 128);   // a box holds tpt tokens x G heads
        for (int w = 0; w < NT; ++w)
          for (int h = 0; h < nslab; ++h)
            tma_load_4d(q_s + w * C::Q_BYTES + h * BM * 128, &map_q, q_full, h * 64, 0, g.kvh, g.tok0 + w * tpt);
        const int last_own = FORM != SHARED ? max(min((seq_pos + g.tok0 - seq_start + g.n_tok - s.prefix_len - 1) / PAGE, s.width - 1), 0) : 0;
        for (int j = 0; j < g.nb; ++j, ++it) {
          const int st = it % C::ST;
          int row0[KB / PAGE];
#pragma unroll
          for (int half = 0; half < KB / PAGE; ++half) {   // a block's second page may lie behind the last: those keys are masked
            int page;
            if (FORM == SHARED || j < g.n_shared) page = s.prefix_pages[min((g.block0 + j) * (KB / PAGE) + half, last_shared)];
            else page = s.table[(size_t)seq * s.ld_table + min((j - g.n_shared) * (KB / PAGE) + half, last_own)];
            row0[half] = (max(page, 0) * s.nkv + g.kvh) * PAGE;
          }
          if (it >= C::ST && !(ok = mbar_wait(k_empty + 8 * st, (it / C::ST - 1) & 1, status, 41))) break;
          jb::mbar_expect_tx(k_full + 8 * st, nslab * KB * 128);
#pragma unroll
          for (int half = 0; half < KB / PAGE; ++half)
            for (int h = 0; h < nslab; ++h)
              jb::tma_load_2d(k_s + st * C::KV_BYTES + h * KB * 128 + half * PAGE * 128, &map_k, k_full + 8 * st, h * 64, row0[half]);
          if (it >= C::ST && !(ok = mbar_wait(v_empty + 8 * st, (it / C::ST - 1) & 1, status, 41))) break;
          jb::mbar_expect_tx(v_full + 8 * st, nslab * KB * 128);
#pragma unroll
          for (int half = 0; half < KB / PAGE; ++half)
            for (int h = 0; h < nslab; ++h)
              jb::tma_load_2d(v_s + st * C::KV_BYTES + h * KB * 128 + half * PAGE * 128, &map_v, v_full + 8 * st, h * 64, row0[half]);
        }
      }
    }
  } else if (warp == 1 && C::SPLIT) {
    if (elected()) {
      const uint32_t idesc_s = jb::instr_desc_bf16(KB), idesc_o = jb::instr_desc_bf16((s.hd + 15) & ~15) | (1u << 16);   // values: MN-major
      bool ok = true;
      int begun = 0, scored[2] = {0, 0}, weighed[2] = {0, 0};   // blocks of the segments before; each group's scored, weighed
      for (int at = flat_begin, turn = 0; at < flat_end && ok; ++turn) {
        const Segment g = segment(at);
        if (g.nb == 0 || !(ok = mbar_wait(q_full, turn & 1, status, 42))) break;
        auto scores = [&](int j) -> bool {
          const int st = (begun + j) % C::ST, w = j & 1, b = 2 * w + (w ? scored[1]++ : scored[0]++) % 2;
          if (!mbar_wait(k_full + 8 * st, (begun + j) / C::ST & 1, status, 42)) return false;
          jb::tc_fence_after();
#pragma unroll
          for (int h = 0; h < C::SLABS; ++h) {
            const uint64_t a = jb::smem_desc_sw128(q_s + h * BM * 128), k = jb::smem_desc_sw128(k_s + st * C::KV_BYTES + h * KB * 128);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              if (h * 64 + ks * 16 < s.hd) jb::umma_bf16(tmem + b * KB, a + 2 * ks, k + 2 * ks, idesc_s, (h | ks) ? 1u : 0u);
          }
          jb::umma_commit(s_full(b));
          jb::umma_commit(k_empty + 8 * st);
          return true;
        };
        ok = scores(0) && (g.nb == 1 || scores(1));
        for (int j = 0; j < g.nb && ok; ++j) {
          const int st = (begun + j) % C::ST, w = j & 1, i = w ? weighed[1]++ : weighed[0]++, b = 2 * w + i % 2;
          if (j + 2 < g.nb) ok = scores(j + 2);                // (where this group's weights of two blocks ago have been used)
          ok = ok && mbar_wait(v_full + 8 * st, (begun + j) / C::ST & 1, status, 42);
          if (ok && j == 0 && turn > 0) ok = mbar_wait(o_free(0), (turn - 1) & 1, status, 42);
          if (!ok || !(ok = mbar_wait(p_full(b), i / 2 & 1, status, 42))) break;
          jb::tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < KB / 16; ++ks)
            umma_ts(tmem + C::SB * KB + w * HDC, tmem + b * KB + ks * 8, desc_mn_sw128(v_s + st * C::KV_BYTES + ks * 2048, KB * 128, 1024),
                    idesc_o, j > 1 || ks > 0 ? 1u : 0u);
          jb::umma_commit(o_full(w));
          jb::umma_commit(v_empty + 8 * st);
          if (j == g.nb - 1) jb::umma_commit(o_done(0));
        }
        begun += g.nb;
      }
    }
  } else if (warp == 1) {
    if (elected()) {
      const uint32_t idesc_s = jb::instr_desc_bf16(KB);
      const uint32_t idesc_o = jb::instr_desc_bf16((s.hd + 15) & ~15) | (1u << 16);   // values: MN-major
      auto issue_s = [&](int w, int it) -> bool {
        const int st = it & 1, b = NT == 2 ? w : it & 1;
        if (!mbar_wait(k_full + 8 * st, (it >> 1) & 1, status, 42)) return false;
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
      int at = flat_begin;
      Segment g = segment(at);
      int n = 0, j = 0, turn = 0;                              // blocks of the segment, the next one of them, segments so far
      bool ok = g.nb > 0 && mbar_wait(q_full, 0, status, 42);
      n = g.nb;
      for (int w = 0; w < NT && ok; ++w) ok = issue_s(w, 0);
      for (int it = 0; ok; ++it) {
        const int st = it & 1;
        const bool last = j == n - 1, more = !last || at < flat_end;
        bool fresh_q = last && more;                           // the next block is the first of another segment
        if (NT == 1 && more) {
          if (fresh_q) ok = mbar_wait(q_full, (turn + 1) & 1, status, 42);
          ok = ok && issue_s(0, it + 1);
        }
        for (int w = 0; w < NT && ok; ++w) {
          const int b = NT == 2 ? w : it & 1;
          if (w == 0) ok = mbar_wait(v_full + 8 * st, (it >> 1) & 1, status, 42);
          if (ok && j == 0 && turn > 0) ok = mbar_wait(o_free(w), (turn - 1) & 1, status, 42);
#pragma unroll
          for (int c = 0; c < C::CHUNKS && ok; ++c) {
            ok = mbar_wait(c < C::CHUNKS - 1 ? p_half(b) : p_full(b), (NT == 2 ? it : it >> 1) & 1, status, 42);
            if (!ok) break;
            jb::tc_fence_after();
#pragma unroll
            for (int k2 = 0; k2 < 4; ++k2) {                    // 32 keys of each of a block's halves (with 64 keys a block: all)
              const int ks = (k2 >> 1) * (KB / 32) + c * 2 + (k2 & 1);
              umma_ts(tmem + 2 * KB + w * HDC, tmem + b * KB + ks * 8, desc_mn_sw128(v_s + st * C::KV_BYTES + ks * 2048, KB * 128, 1024),
                      idesc_o, (j | ks) ? 1u : 0u);
            }
          }
          if (!ok) break;
          jb::umma_commit(o_full(w));
          if (last) jb::umma_commit(o_done(w));
          if (w == NT - 1) jb::umma_commit(v_empty + 8 * st);
          if (NT == 2 && more) {
            if (fresh_q) ok = mbar_wait(q_full, (turn + 1) & 1, status, 42), fresh_q = false;
            ok = ok && issue_s(w, it + 1);
          }
        }
        if (!more) break;
        ++j;
        if (last) {
          g = segment(at);
          n = g.nb, j = 0, ++turn;
        }
      }
    }
  } else {
    // two warps have the same 32 rows, each half of a block's keys (SPLIT: every second block of keys, of 64), and half of O's columns
    const int w = (warp - 2) >> 3, quarter = warp & 3, half = (warp - 2) >> 2 & 1, row = quarter * 32 + lane, pair = 1 + w * 4 + quarter;
    constexpr int KH = C::SPLIT ? KB : KB / 2, DH = HDC / 2;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16), o_col = C::SB * KB + w * HDC;
    float* mine = swap + (w * 2 + half) * BM + row;
    const float* other = swap + (w * 2 + (half ^ 1)) * BM + row;
    // The two say to each other that a row's maximum has grown, or that a wait has run out: then both leave, behind a barrier that
    // they share.  (A value is read before its place is written again: the writer has passed another barrier with the reader.)
    int* stop = gave_up + w * 4 + quarter;
    bool ok = true, both = true;
    int it = 0, turn = 0;
    auto meet = [&](float value) {
      *mine = value;
      if (!ok) *stop = 1;
      pair_sync(pair);
      both = *(volatile int*)stop == 0;
      return *other;
    };
    for (int at = flat_begin; at < flat_end && both; ++turn) {
      const Segment g = segment(at);
      if (g.n_tok <= 0 && FORM != SHARED) break;
      const int tl = w * tpt + row / G, token = g.tok0 + tl, head = g.kvh * G + row % G;
      const bool valid = row < tpt * G && tl < g.n_tok;        // rows past tpt * G belong to no token
      int see_shared = 0, see_own = 0;                         // keys that the row sees, counted from its half's first
      if (valid) {
        const int see = (FORM == SHARED ? s.positions[token] : seq_pos + token - seq_start) + 1;
        see_shared = min(see, s.prefix_len) - g.block0 * KB - (C::SPLIT ? 0 : half * KH);
        see_own = see - s.prefix_len - (C::SPLIT ? 0 : half * KH);
      }
      float m_ref = -CUDART_INF_F, l = 0.0f;
      float weight[2] = {1.0f, 0.0f};                          // SPLIT: of the groups' O, once they are joined
      if constexpr (C::SPLIT) {
        const uint32_t my_o = lane_addr + o_col + half * HDC;
        for (int j = half; j < g.nb; j += 2, ++it) {
          const int b = 2 * half + (it & 1);
          const uint32_t s_at = lane_addr + b * KB;
          ok = __all_sync(0xffffffffu, mbar_wait(s_full(b), (it >> 1) & 1, status, 43));
          if (!ok) break;
          jb::tc_fence_after();
          uint32_t sr[KH];
#pragma unroll
          for (int c0 = 0; c0 < KH; c0 += 16) tmem_ld16(s_at + c0, sr + c0);
          jb::tmem_ld_wait();
          const int see = j < g.n_shared ? see_shared - j * KB : see_own - (j - g.n_shared) * KB;
          if (see < KH) {
#pragma unroll
            for (int c = 0; c < KH; ++c)
              if (c >= see) sr[c] = 0xff800000u;   // -inf
          }
          const float mx = row_max<KH>(sr) * s.scale_log2;
          if (__any_sync(0xffffffffu, mx > m_ref + RESCALE_LOG2 || (m_ref == -CUDART_INF_F && mx > -CUDART_INF_F))) {
            const float m_new = fmaxf(m_ref, mx);
            if (j > 1) {
              ok = __all_sync(0xffffffffu, mbar_wait(o_full(half), (it - 1) & 1, status, 43));
              if (!ok) break;
              jb::tc_fence_after();
              const float corr = m_new == -CUDART_INF_F ? 1.0f : exp2f(m_ref - m_new);
#pragma unroll
              for (int c0 = 0; c0 < HDC; c0 += 16) {
                if (c0 >= s.hd) break;
                uint32_t r[16];
                tmem_ld16(my_o + c0, r);
                jb::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * corr);
                tmem_st16(my_o + c0, r);
              }
              l *= corr;
            }
            m_ref = m_new;
          }
          l += exp_pack_sum<KH, false>(sr, s.scale_log2, m_ref == -CUDART_INF_F ? 0.0f : -m_ref);
#pragma unroll
          for (int c0 = 0; c0 < KH / 2; c0 += 16) tmem_st16(s_at + c0, sr + c0);
          tmem_st_wait();
          jb::tc_fence_before();
          __syncwarp();
          if (lane == 0) jb::mbar_arrive(p_full(b));
        }
        if (ok && g.nb > 0) ok = __all_sync(0xffffffffu, mbar_wait(o_done(0), turn & 1, status, 43));
        // both groups' sums, joined as those of any two sets of keys
        const float their_m = meet(m_ref);
        if (!both) break;
        pair_sync(pair);                // (the place is read before it is written again)
        const float their_l = meet(l);
        if (!both) break;
        pair_sync(pair);
        const float top = fmaxf(m_ref, their_m), ref = top == -CUDART_INF_F ? 0.0f : top;
        weight[half] = exp2f(m_ref - ref), weight[half ^ 1] = exp2f(their_m - ref);
        l = half == 0 ? fmaf(l, weight[0], their_l * weight[1]) : fmaf(their_l, weight[0], l * weight[1]);
        m_ref = top;
        jb::tc_fence_after();
      }
      // 16 columns of O
      auto load_o = [&](int c0, uint32_t* r) {
        tmem_ld16(lane_addr + o_col + c0, r);   // warp-wide: rows without a token load too
        if constexpr (C::SPLIT) {
          if (g.nb > 1) {
            uint32_t second[16];
            tmem_ld16(lane_addr + o_col + HDC + c0, second);
            jb::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i)
              r[i] = __float_as_uint(fmaf(__uint_as_float(r[i]), weight[0], __uint_as_float(second[i]) * weight[1]));
            return;
          }
        }
        jb::tmem_ld_wait();
      };
      for (int j = 0; j < g.nb && !C::SPLIT; ++j, ++it) {
        const int b = NT == 2 ? w : it & 1;
        const uint32_t s_at = lane_addr + b * KB;
        ok = __all_sync(0xffffffffu, ok && mbar_wait(s_full(b), (NT == 2 ? it : it >> 1) & 1, status, 43));
        jb::tc_fence_after();
        uint32_t sr[KH];
#pragma unroll
        for (int c0 = 0; c0 < KH; c0 += 16) tmem_ld16(s_at + half * KH + c0, sr + c0);
        jb::tmem_ld_wait();
        const int see = j < g.n_shared ? see_shared - j * KB : see_own - (j - g.n_shared) * KB;
        if (see < KH) {
#pragma unroll
          for (int c = 0; c < KH; ++c)
            if (c >= see) sr[c] = 0xff800000u;   // -inf
        }
        float mx = row_max<KH>(sr) * s.scale_log2;
        // behind this barrier both halves have their scores, and P may go where scores lie.  Loads and stores of tensor memory
        // are warp-wide: the two warps rescale together if any of their rows has to
        const bool grow = mx > m_ref + RESCALE_LOG2 || (m_ref == -CUDART_INF_F && mx > -CUDART_INF_F);
        jb::tc_fence_before();
        const bool any = pair_any(pair, grow || !ok);
        jb::tc_fence_after();
        if (any) {
          mx = fmaxf(mx, meet(mx));   // the row's, over both halves
          if (!both) break;
          const float m_new = fmaxf(m_ref, mx);
          if (j > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(o_full(w), (it - 1) & 1, status, 43));
            if (!ok) continue;
            jb::tc_fence_after();
            const float corr = m_new == -CUDART_INF_F ? 1.0f : exp2f(m_ref - m_new);
#pragma unroll
            for (int c0 = 0; c0 < DH; c0 += 16) {
              if (half * DH + c0 >= s.hd) break;
              uint32_t r[16];
              tmem_ld16(lane_addr + o_col + half * DH + c0, r);
              jb::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * corr);
              tmem_st16(lane_addr + o_col + half * DH + c0, r);
            }
            tmem_st_wait();
            l *= corr;
          }
          m_ref = m_new;
        }
        // 32 keys of each half at a time: the product with the first ones' values runs while the others' weights are made
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c) {
          l += exp_pack_sum<32, NT == 2>(sr + 32 * c, s.scale_log2, m_ref == -CUDART_INF_F ? 0.0f : -m_ref);
          tmem_st16(s_at + half * (KH / 2) + 16 * c, sr + 32 * c);
          tmem_st_wait();
          jb::tc_fence_before();
          __syncwarp();
          if (lane == 0) jb::mbar_arrive(c < C::CHUNKS - 1 ? p_half(b) : p_full(b));
        }
      }
      if constexpr (!C::SPLIT) {
        if (!both) break;
        if (ok && g.nb > 0) ok = __all_sync(0xffffffffu, mbar_wait(o_done(w), turn & 1, status, 43));
        const float theirs = meet(l);   // the row's sum over both halves
        if (!both) break;
        l = half == 0 ? l + theirs : theirs + l;
        pair_sync(pair);                // (the place is read before it is written again)
        jb::tc_fence_after();
      }
      const size_t place = (size_t)token * s.nh + head, all = (size_t)s.T * s.nh;
      if (FORM == SHARED || (FORM == OWN && parts.most > 1)) {
        const size_t item = (FORM == SHARED ? g.slot : parts.most) * all + place;
        if (valid && half == 0) part_ml[item] = make_float2(m_ref, l);
#pragma unroll
        for (int c1 = 0; c1 < DH; c1 += 16) {
          const int c0 = half * DH + c1;
          if (c0 >= s.hd) break;
          uint32_t r[16];
          load_o(c0, r);
          if (FORM == OWN && g.nb == 0) {         // (no product has written there)
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = 0u;
          }
          if (valid) store8(part_o + item * s.hd + c0, r);
          if (valid && c0 + 8 < s.hd) store8(part_o + item * s.hd + c0 + 8, r + 8);
        }
        jb::tc_fence_before();
        __syncwarp();
        if (lane == 0) jb::mbar_arrive(o_free(w));
      } else {
        // the one part over the prefix weighs in (OWN)
        const int slots = FORM == OWN && valid ? parts.most : 0;
        if (FORM == OWN) jb::pdl_wait();
        float top = m_ref;
        for (int i = 0; i < slots; ++i) top = fmaxf(top, part_ml[i * all + place].x);
        const float ref = top == -CUDART_INF_F ? 0.0f : top, own_weight = exp2f(m_ref - ref);
        l *= own_weight;
        for (int i = 0; i < slots; ++i) {
          const float2 ml = part_ml[i * all + place];
          l = fmaf(exp2f(ml.x - ref), ml.y, l);
        }
        const float inv = top == -CUDART_INF_F ? 0.0f : 1.0f / l;   // (a row that sees nothing)
        bool finite = true;
#pragma unroll
        for (int c1 = 0; c1 < DH; c1 += 16) {
          const int c0 = half * DH + c1;
          if (c0 >= s.hd) break;
          uint32_t r[16];
          if (g.nb > 0) load_o(c0, r);
          float v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = g.nb > 0 ? __uint_as_float(r[i]) * own_weight : 0.0f;
          if constexpr (FORM == OWN) {
            for (int i = 0; i < slots; ++i) {
              const float f = exp2f(part_ml[i * all + place].x - ref);
              float more[16];
              load8(part_o + (i * all + place) * s.hd + c0, more);
              if (c0 + 8 < s.hd) load8(part_o + (i * all + place) * s.hd + c0 + 8, more + 8);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (e < 8 || c0 + 8 < s.hd) v[e] = fmaf(f, more[e], v[e]);
            }
          }
          uint32_t p[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x = v[2 * i] * inv, y = v[2 * i + 1] * inv;
            finite = finite && (c0 + 2 * i >= s.hd || (isfinite(x) && isfinite(y)));
            p[i] = pack_bf16(x, y);
          }
          if (valid) {
            *reinterpret_cast<uint4*>(out + place * s.hd + c0) = make_uint4(p[0], p[1], p[2], p[3]);
            if (c0 + 8 < s.hd) *reinterpret_cast<uint4*>(out + place * s.hd + c0 + 8) = make_uint4(p[4], p[5], p[6], p[7]);
          }
        }
        // a row that is not finite is made once more by itself, by its first half's warp, when both halves have written
        finite = meet(finite ? 0.0f : 1.0f) == 0.0f && finite;
        unsigned again = half == 0 ? __ballot_sync(0xffffffffu, valid && !finite) : 0u;
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
  if (FORM == OWN && (parts.most == 1 || blockIdx.x + blockIdx.y == 0)) jb::pdl_wait();   // (see own_kernel's end)
  __syncthreads();
  if (warp == 1) {
    jb::tc_fence_after();
    jb::tmem_dealloc<C::COLS>(tmem);
  }
}

// ---------------------------------------------------------------------------
// bfloat16: each sequence's own pages, by warp-level products.  The work is a flat list: sequence after sequence, its (kv head, 16 rows)
// pairs, their tiles of 32 keys.  Every warp has an even, consecutive share of it and works by itself: the copy engine brings its
// tiles (128-byte swizzle) into a ring of its own, ahead across the ends of rows, the rows' queries stay in registers as the
// products take them, and where a row's keys end (or the share does) the sums go out as a partial result.  How many a row has is
// written beside (own_count).  A block of its own for every row waited for the longest row, and for what it had to fetch before
// its first key: 256 sequences of 3 to 2,500 keys moved 2.8 TB/s; by shares 5.2 (359 MB in 69 us, the machine to itself).  Warp-level
// products, as the 16 rows that a sequence has are an eighth of a tensor-core tile.  The count is one of each (token, query head): 16
// rows end inside a token where the heads of a group do not divide them, and its other heads are then cut at other places.
// ---------------------------------------------------------------------------
constexpr int OWN_WARPS = 4, OWN_THREADS = 32 * OWN_WARPS, OWN_KEYS = 32, OWN_HALVES = PAGE / OWN_KEYS;

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
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
  static constexpr int SLABS = HDC / 64, SLAB = OWN_KEYS * 128;            // bytes of 64 numbers of a warp's keys
  static constexpr int TILE = SLABS * SLAB, STAGE = 2 * TILE;              // keys, values
  static constexpr int RING = OWN_WARPS * STAGES * STAGE;
  static constexpr int SMEM = RING + OWN_WARPS * STAGES * 16;
};

// A place of the list: the tile, and what its rows are.
struct Cursor {
  int seq, kvh, rb, tile;           // sequence; kv head, block of 16 rows; tile of the row's keys
  int tiles, row_blocks, start, q_len;
  int shared;                       // tiles of the prefix in front, where the list holds them
  int most;                         // tiles of own keys at most
};
// What sequence `seq` adds to the list: every row has a tile, also one that sees no key of its own.  No more than `most` behind the
// prefix, by the caller's bound of the lengths: the places for partial results are counted by it, whatever kv_len says.
__device__ __forceinline__ void look_up(const Step& s, int seq, int shared, int most, Cursor& c) {
  c.seq = seq, c.start = s.q_start[seq], c.q_len = s.q_start[seq + 1] - c.start;
  c.row_blocks = c.q_len > 0 ? (c.q_len * (s.nh / s.nkv) + 15) / 16 : 0;
  c.shared = shared, c.most = most;
  c.tiles = shared + min(max((s.kv_len[seq] - s.prefix_len + OWN_KEYS - 1) / OWN_KEYS, 1), most);
}
__device__ __forceinline__ int places(const Step& s, const Cursor& c) { return s.nkv * c.row_blocks * c.tiles; }
__device__ __forceinline__ void step_on(const Step& s, Cursor& c) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.rb < c.row_blocks) return;
  c.rb = 0;
  if (++c.kvh < s.nkv) return;
  c.kvh = 0;
  do {
    if (c.seq + 1 >= s.n_seqs) return;   // (behind the list's end: nobody goes there)
    look_up(s, c.seq + 1, c.shared, c.most, c);
  } while (c.row_blocks == 0);
}

template <int HDC, int STAGES>
__global__ void __launch_bounds__(OWN_THREADS) own_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                          const bf16* __restrict__ q, float* __restrict__ part_o, float2* __restrict__ part_ml,
                                                          int* __restrict__ own_count, const Step s, int first_slot, int after_prefix,
                                                          int shared, int most, int fewest, int* __restrict__ status) {
  typedef Own<HDC, STAGES> C;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = (uint64_t*)(smem + C::RING);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, hd = s.hd, G = s.nh / s.nkv;
  const uint32_t ring = jb::smem_u32(smem) + warp * STAGES * C::STAGE, bar = jb::smem_u32(full + warp * STAGES * 2);
  if (lane == 0) {
    for (int i = 0; i < STAGES * 2; ++i) jb::mbar_init(bar + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (!after_prefix) jb::pdl_wait();
  jb::pdl_launch_dependents();
  // ---- the list's length, and this warp's share ----
  Cursor c{};
  const int chunk = (s.n_seqs + 31) / 32, seq0 = min(lane * chunk, s.n_seqs), seq1 = min(seq0 + chunk, s.n_seqs);
  int mine = 0;
#pragma unroll 4
  for (int i = seq0; i < seq1; ++i) {
    Cursor x;
    look_up(s, i, shared, most, x);
    mine += places(s, x);
  }
  int up = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += t;
  }
  const int total = __shfl_sync(0xffffffffu, up, 31), worker = blockIdx.x * OWN_WARPS + warp;
  const int per = max(fewest, (total + (int)gridDim.x * OWN_WARPS - 1) / ((int)gridDim.x * OWN_WARPS));
  const int begin = min(worker * per, total), end = min(begin + per, total);
  if (begin < end) {
    const int owner = __ffs(__ballot_sync(0xffffffffu, begin < up)) - 1;
    int before = __shfl_sync(0xffffffffu, up - mine, owner);
    for (int i = owner * chunk;; ++i) {
      look_up(s, i, shared, most, c);
      const int n = places(s, c);
      if (begin < before + n) break;
      before += n;
    }
    const int y = (begin - before) / c.tiles;
    c.tile = (begin - before) - y * c.tiles, c.kvh = y / c.row_blocks, c.rb = y - c.kvh * c.row_blocks;
  }
  const uint64_t policy = jb::read_once_policy();
  const int nslab = (hd + 63) / 64;
  Cursor ahead = c;
  int asked = begin;
  // (a tile's page is looked up a turn before it is asked for, or every turn would wait for memory)
  auto page_of = [&](const Cursor& x) {
    if (x.tile < x.shared) return s.prefix_pages[x.tile / OWN_HALVES];
    return s.width > 0 ? s.table[(size_t)x.seq * s.ld_table + (x.tile - x.shared) / OWN_HALVES] : 0;
  };
  int page = begin < end ? page_of(ahead) : 0;
  // Keys and values of a tile have a barrier each: with one stage the next keys are on their way while this tile's softmax and the
  // values' product run, the next values during the scores.
  auto issue = [&](int what) {   // 0: the keys of the next tile that has not been asked for; 1: its values, and on to the one behind
    const int st = (asked - begin) % STAGES;
    if (elected()) {
      const int half = (ahead.tile < ahead.shared ? ahead.tile : ahead.tile - ahead.shared) % OWN_HALVES;
      const int row = (max(page, 0) * s.nkv + ahead.kvh) * PAGE + half * OWN_KEYS;
      const uint32_t at = ring + st * C::STAGE + what * C::TILE, full_at = bar + 16 * st + 8 * what;
      jb::mbar_expect_tx(full_at, nslab * C::SLAB);
      for (int h = 0; h < nslab; ++h) jb::tma_load_2d(at + h * C::SLAB, what ? &map_v : &map_k, full_at, h * 64, row, policy);
    }
    __syncwarp();
    if (what == 0) return;
    ++asked;
    if (asked < end) {
      step_on(s, ahead);
      page = page_of(ahead);
    }
  };
  for (int i = 0; i < STAGES; ++i)
    if (asked < end) issue(0), issue(1);
  // the rows' queries as the A operand of the products: lane (g, c) has rows g and g + 8, numbers 2 c, 2 c + 1 and 8 behind of every 16
  uint32_t qa[HDC / 16][4];
  float m[2], l[2], o[HDC / 8][4];
  int see_row[2];
  bool ok = true;
  for (int i = begin; i < end; ++i) {
    if (i == begin || c.tile == 0) {
      const int kvh = c.kvh, row0 = c.rb * 16, n_rows = min(16, c.q_len * G - row0);
      const int first_pos = s.kv_len[c.seq] - c.q_len;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = (lane >> 2) + 8 * r, token = (row0 + row) / G, head = kvh * G + (row0 + row) % G;
        const bool valid = row < n_rows;
        see_row[r] = valid ? first_pos + token + 1 : 0;   // keys that the row sees, the prefix's first
        m[r] = -CUDART_INF_F, l[r] = 0.0f;
        const bf16* src = q + ((size_t)(c.start + (valid ? token : 0)) * s.nh + head) * hd + 2 * (lane & 3);
#pragma unroll
        for (int ks = 0; ks < HDC / 16; ++ks)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            qa[ks][r + 2 * half] = valid && ks * 16 + half * 8 < hd ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + half * 8) : 0u;
      }
#pragma unroll
      for (int j = 0; j < HDC / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    }
    const int turn = i - begin, st = turn % STAGES;
    ok = mbar_wait(bar + 16 * st, (turn / STAGES) & 1, status, 53);
    if (__any_sync(0xffffffffu, !ok)) break;
    const uint32_t k_t = ring + st * C::STAGE, v_t = k_t + C::TILE;
    float x[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < HDC / 16; ++ks) {
      if (ks * 16 >= hd) break;
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        uint32_t b[4];
        const int key = j * 8 + (lane & 7) + ((lane >> 4) << 3), piece = (ks % 4) * 2 + ((lane >> 3) & 1);
        ldmatrix_x4(b, k_t + (ks / 4) * C::SLAB + key * 128 + ((piece ^ (key & 7)) << 4));
        mma_bf16(x[j], qa[ks], b[0], b[1]);
        mma_bf16(x[j + 1], qa[ks], b[2], b[3]);
      }
    }
    __syncwarp();   // the warp is done with the keys
    if (asked < end) issue(0);
    float mx[2] = {-CUDART_INF_F, -CUDART_INF_F}, corr[2], ref[2];
    const bool of_prefix = c.tile < c.shared;
    const int key0 = (of_prefix ? c.tile : c.tile - c.shared) * OWN_KEYS + 2 * (lane & 3);
    int limit[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) limit[r] = of_prefix ? min(see_row[r], s.prefix_len) : min(see_row[r] - s.prefix_len, s.width * PAGE);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[j][e] = key0 + j * 8 + (e & 1) < limit[e >> 1] ? x[j][e] * s.scale_log2 : -CUDART_INF_F;
        mx[e >> 1] = fmaxf(mx[e >> 1], x[j][e]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      const float m_new = fmaxf(m[r], mx[r]);
      ref[r] = m_new == -CUDART_INF_F ? 0.0f : m_new;
      corr[r] = fast_exp2(m[r] - ref[r]);
      m[r] = m_new;
      l[r] *= corr[r];
    }
#pragma unroll
    for (int j = 0; j < HDC / 8; ++j) o[j][0] *= corr[0], o[j][1] *= corr[0], o[j][2] *= corr[1], o[j][3] *= corr[1];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[j][e] = fast_exp2(x[j][e] - ref[e >> 1]);
        l[e >> 1] += x[j][e];
      }
    ok = mbar_wait(bar + 16 * st + 8, (turn / STAGES) & 1, status, 53);
    if (__any_sync(0xffffffffu, !ok)) break;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const uint32_t a[4] = {pack_bf16(x[2 * kk][0], x[2 * kk][1]), pack_bf16(x[2 * kk][2], x[2 * kk][3]),
                             pack_bf16(x[2 * kk + 1][0], x[2 * kk + 1][1]), pack_bf16(x[2 * kk + 1][2], x[2 * kk + 1][3])};
#pragma unroll
      for (int j = 0; j < HDC / 8; j += 2) {
        if (j * 8 >= hd) break;
        uint32_t b[4];
        const int key = kk * 16 + (lane & 15), piece = j % 8 + (lane >> 4);
        ldmatrix_x4_trans(b, v_t + (j / 8) * C::SLAB + key * 128 + ((piece ^ (key & 7)) << 4));
        mma_bf16(o[j], a, b[0], b[1]);
        mma_bf16(o[j + 1], a, b[2], b[3]);
      }
    }
    __syncwarp();   // ... and with the values
    if (asked < end) issue(1);
    if (i + 1 == end || c.tile + 1 == c.tiles) {   // the row's keys end here, or the share does
      const int place = i - c.tile, first = place / per, slot = worker - first;
      const int kvh = c.kvh, row0 = c.rb * 16, n_rows = min(16, c.q_len * G - row0);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        const int row = (lane >> 2) + 8 * r, token = c.start + (row0 + row) / G, head = kvh * G + (row0 + row) % G;
        if (row >= n_rows) continue;
        const size_t item = ((size_t)(first_slot + slot) * s.T + token) * s.nh + head;
        if ((lane & 3) == 0) {
          part_ml[item] = make_float2(m[r], l[r]);
          if (slot == 0) own_count[token * s.nh + head] = (place + c.tiles - 1) / per - first + 1;
        }
#pragma unroll
        for (int j = 0; j < HDC / 8; ++j)
          if (j * 8 < hd) *reinterpret_cast<float2*>(part_o + item * hd + j * 8 + 2 * (lane & 3)) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
      }
    }
    if (i + 1 < end) step_on(s, c);
  }
  // Who waits for this launch has to have waited for the one before it: one block sees to that.  (All of them waiting held their places
  // on the multiprocessors until the prefix was done, and the blocks behind them had none: 256 long sequences 144 us.)
  if (after_prefix && blockIdx.x == 0) jb::pdl_wait();
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// q's tiles (null: none are wanted), and the pages in boxes of `keys` rows
bool make_maps(CUtensorMap* mq, CUtensorMap* mk, CUtensorMap* mv, const void* q, const void* k, const void* v, const Step& s, int n_pages,
               int keys) {
  static jb::EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess)
      return false;
    fn = (jb::EncodeTiledFn)p;
  }
  const cuuint32_t el[4] = {1, 1, 1, 1};
  if (mq) {
    const cuuint64_t G = s.nh / s.nkv, hd = s.hd;
    const cuuint64_t dims[4] = {hd, G, (cuuint64_t)s.nkv, (cuuint64_t)s.T}, strides[3] = {hd * 2, G * hd * 2, (cuuint64_t)s.nh * hd * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)G, 1, (cuuint32_t)(BM / G)};
    if (fn(mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(q), dims, strides, box, el, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  }
  for (int which = 0; which < 2; ++which) {
    const cuuint64_t dims[2] = {(cuuint64_t)s.hd, (cuuint64_t)n_pages * s.nkv * PAGE}, strides[1] = {(cuuint64_t)s.hd * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)keys};
    if (fn(which ? mv : mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(which ? v : k), dims, strides, box, el,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  }
  return true;
}

template <int HDC, int NT, int KB, Form FORM>
cudaError_t tc_go(dim3 grid, cudaStream_t stream, const CUtensorMap* maps, const bf16* q, const bf16* k, const bf16* v, bf16* out,
                  float* part_o, float2* part_ml, const Step& s, const Slots& parts, int* status) {
  typedef Tc<HDC, NT, KB> C;
  static bool configured = false;
  if (!configured) {
    cudaError_t e = set_up(prefix_tc_kernel<HDC, NT, KB, FORM>, C::SMEM);
    if (e != cudaSuccess) return e;
    configured = true;
  }
  jb::Launch cfg(grid, dim3(C::THREADS), C::SMEM, stream);
  return cudaLaunchKernelEx(&cfg.c, prefix_tc_kernel<HDC, NT, KB, FORM>, maps[0], maps[1], maps[2], q, k, v, out, part_o, part_ml, s, parts,
                            status);
}
template <Form FORM>
cudaError_t tc_pick(int nt, dim3 grid, cudaStream_t stream, const CUtensorMap* maps, const bf16* q, const bf16* k, const bf16* v, bf16* out,
                    float* part_o, float2* part_ml, const Step& s, const Slots& parts, int* status) {
#define JB_GO(HDC, NT, KB) return tc_go<HDC, NT, KB, FORM>(grid, stream, maps, q, k, v, out, part_o, part_ml, s, parts, status)
  if (s.hd > 128) JB_GO(256, 1, 64);
  if (s.hd > 64 && nt == 2) JB_GO(128, 2, 128);
  if (s.hd > 64) JB_GO(128, 1, 128);
  if (nt == 2) JB_GO(64, 2, 128);
  JB_GO(64, 1, 64);
#undef JB_GO
}

template <int HDC, int STAGES>
cudaError_t own_go(int blocks, cudaStream_t stream, const CUtensorMap* maps, const bf16* q, float* part_o, float2* part_ml, int* own_count,
                   const Step& s, int first_slot, int after_prefix, int shared, int most, int fewest, int* status) {
  typedef Own<HDC, STAGES> C;
  static bool configured = false;
  if (!configured) {
    cudaError_t e = set_up(own_kernel<HDC, STAGES>, C::SMEM);
    if (e != cudaSuccess) return e;
    configured = true;
  }
  jb::Launch cfg(dim3(blocks), dim3(OWN_THREADS), C::SMEM, stream);
  return cudaLaunchKernelEx(&cfg.c, own_kernel<HDC, STAGES>, maps[0], maps[1], q, part_o, part_ml, own_count, s, first_slot, after_prefix,
                            shared, most, fewest, status);
}

}  // namespace

// q, out [T, nh hd], caches [n_pages, nkv, 64, hd], all bfloat16.  tiles: row tiles of a block, 1 or 2 (one for heads of more than 128
// numbers).  shared_per > 0: the prefix for all rows together by blocks of that many key blocks each, which cut a row's keys into at
// most `most` ranges.  own_tiles: own keys by tiles of a sequence each, else by the warps of own_ctas blocks, which get no less than
// `fewest` tiles of 32 keys each, so that a row has at most own_most partial results; with the prefix's keys, where nobody walks those
// apart.  scratch: floats [most + own_most][T][nh][hd], then [..][T][nh][2], then T nh whole numbers (own_most 1 with own_tiles and
// several ranges).
// tensors, sizes: host memory, see Tensors and Sizes.
JB_EXPORT int jb_attention_prefix_bf16(const void* tensors, const void* sizes, int* status, cudaStream_t stream) {
  const Tensors& t = *(const Tensors*)tensors;
  const Sizes& z = *(const Sizes*)sizes;
  const void *q = t.q, *k_cache = t.k_cache, *v_cache = t.v_cache;
  void* out = t.out;
  float* scratch = t.scratch;
  const int prefix_len = z.prefix_len, T = z.T, n_pages = z.n_pages, n_seqs = z.n_seqs, nh = z.nh, nkv = z.nkv, hd = z.hd;
  const int page_size = z.page_size, max_q_len = z.max_q_len, max_kv_len = z.max_kv_len, tiles = z.tiles, shared_per = z.shared_per;
  const int most = z.most, own_tiles = z.own_tiles, own_ctas = z.own_ctas, fewest = z.fewest, own_most = z.own_most;
  if (T <= 0 || n_seqs <= 0 || max_q_len <= 0) return 0;
  JB_REFUSE(page_size != PAGE, "attention_prefix: page size %d (need %d)", page_size, PAGE);
  JB_REFUSE(nkv <= 0 || nh % nkv != 0, "attention_prefix: %d heads are not a multiple of %d kv heads", nh, nkv);
  JB_REFUSE(hd <= 0 || hd > 256 || hd % 8 != 0, "attention_prefix: bfloat16 heads of %d numbers (multiples of 8 up to 256)", hd);
  const int G = nh / nkv;
  JB_REFUSE(G > BM, "attention_prefix: %d query heads per kv head are more than %d", G, BM);
  JB_REFUSE(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15, "attention_prefix: operands must be 16-byte aligned");
  JB_REFUSE((long long)n_pages * nkv * PAGE > 0x7fffffffll, "attention_prefix: %d pages of %d heads are more rows than a tensor map counts",
            n_pages, nkv);
  JB_REFUSE(n_seqs > 65535 || prefix_len < 0 || shared_per < 0 || most < 0 || most > 64 || (shared_per > 0) != (most > 0) ||
                (shared_per > 0 && prefix_len == 0),
            "attention_prefix: a prefix of %d tokens in %d ranges of %d key blocks for %d sequences", prefix_len, most, shared_per, n_seqs);
  const Step s{t.prefix_pages, t.block_table, t.q_start, t.kv_len, t.positions, prefix_len, z.ld_table, z.width, T, n_seqs, nh, nkv, hd, z.scale * LOG2E};
  const bf16 *qb = (const bf16*)q, *kb = (const bf16*)k_cache, *vb = (const bf16*)v_cache;
  bf16* ob = (bf16*)out;
  const size_t rows_of_parts = (size_t)(most + own_most) * T * nh;
  float* part_o = scratch;
  float2* ml = (float2*)(scratch + rows_of_parts * hd);
  int* own_count = (int*)(ml + rows_of_parts);
  const int nt = hd > 128 ? 1 : tiles, step = nt * (BM / G), keys = hd > 128 ? 64 : 128;
  Slots parts{0, 0, 0, 1, 1};
  CUtensorMap maps[3];
  if ((shared_per > 0 || own_tiles) && !make_maps(&maps[0], &maps[1], &maps[2], q, k_cache, v_cache, s, n_pages, PAGE)) return JB_ERR_TENSORMAP;
  cudaError_t e = cudaSuccess;
  if (shared_per > 0) {
    int blocks = (prefix_len + keys - 1) / keys;
    const long long items = (long long)((T + step - 1) / step) * nkv;
    // A tile's last range may be shorter than the others, where all of them still run at once: a block that goes from one tile to the
    // next in its range pays queries, result and the start of its products twice.
    const int even = (blocks + shared_per - 1) / shared_per;
    if (shared_per < blocks && items * even <= SMS) blocks = even * shared_per;
    const long long total = items * blocks, ctas = (total + shared_per - 1) / shared_per;
    // a tile's blocks begin anywhere in a range, unless ranges divide them, or are whole tiles
    JB_REFUSE(total > 0x3fffffffll, "attention_prefix: %lld key blocks", total);
    JB_REFUSE((shared_per % blocks == 0 ? 1 : blocks % shared_per == 0 ? blocks / shared_per : (blocks + shared_per - 2) / shared_per + 1) > most,
              "attention_prefix: ranges of %d cut %d key blocks into more than %d", shared_per, blocks, most);
    const int finer = hd <= 64 && nt == 1 ? 2 : 1;             // such a tile's blocks have 64 keys
    parts = Slots{-1, most, blocks * finer, shared_per * finer, step};
    e = tc_pick<SHARED>(nt, dim3((unsigned)ctas), stream, maps, qb, kb, vb, ob, part_o, ml, s, parts, status);
    if (e != cudaSuccess) return (int)e;
  }
  if (own_tiles) {
    const dim3 grid(nkv, T / step + (n_seqs < T ? n_seqs : T));   // no more tiles than that, however the tokens are shared out
    JB_REFUSE(grid.y > 65535, "attention_prefix: %d tokens of %d sequences", T, n_seqs);
    e = shared_per > 0 ? tc_pick<OWN>(nt, grid, stream, maps, qb, kb, vb, ob, part_o, ml, s, parts, status)
                       : tc_pick<WHOLE>(nt, grid, stream, maps, qb, kb, vb, ob, part_o, ml, s, parts, status);
    if (e != cudaSuccess || most <= 1) return (int)e;
    return (int)join_go<bf16>(stream, qb, kb, vb, ob, part_o, ml, nullptr, s, parts, 1);
  }
  // where nobody walks the prefix for all, every sequence's rows walk it with their own keys
  const int shared = shared_per > 0 ? 0 : (prefix_len + OWN_KEYS - 1) / OWN_KEYS;
  const int row_blocks = (max_q_len * G + 15) / 16;
  const int own_tiles_most = (max_kv_len - prefix_len + OWN_KEYS - 1) / OWN_KEYS, tiles_most = shared + (own_tiles_most < 1 ? 1 : own_tiles_most);
  const int in_table = s.width > 0 ? s.width * OWN_HALVES : 1, own_bound = tiles_most - shared < in_table ? tiles_most - shared : in_table;
  JB_REFUSE(own_ctas < 1 || fewest < 1 || own_most > 64 || (tiles_most + fewest - 2) / fewest + 1 > own_most ||
                (long long)n_seqs * nkv * row_blocks * (tiles_most < 1 ? 1 : tiles_most) > 0x3fffffffll,
            "attention_prefix: %d blocks for %d tiles of own keys of %d sequences", own_ctas, tiles_most, n_seqs);
  if (!make_maps(nullptr, &maps[1], &maps[2], q, k_cache, v_cache, s, n_pages, OWN_KEYS)) return JB_ERR_TENSORMAP;
  const int behind = shared_per > 0;
  if (hd > 128) e = own_go<256, 1>(own_ctas, stream, maps + 1, qb, part_o, ml, own_count, s, most, behind, shared, own_bound, fewest, status);
  else if (hd > 64) e = own_go<128, 1>(own_ctas, stream, maps + 1, qb, part_o, ml, own_count, s, most, behind, shared, own_bound, fewest, status);
  else e = own_go<64, 2>(own_ctas, stream, maps + 1, qb, part_o, ml, own_count, s, most, behind, shared, own_bound, fewest, status);
  if (e != cudaSuccess) return (int)e;
  return (int)join_go<bf16>(stream, qb, kb, vb, ob, part_o, ml, own_count, s, parts, own_most);
}
