// Attention of beams over a paged cache, one query token a beam.
//
//   out_i = softmax(q_i K_i' scale) V_i over the first kv_len[i] keys of beam i; scores, maximum and sum in float32, weights
//   rounded to bfloat16 for the product with V, whose accumulators are float32.
//
// Beams of a request hold the same pages up to where they parted.  The rows of a tile are the (beam, query head) pairs of one key
// head, so that a shared page is read once for all beams; behind it every beam's own pages follow, one beam after another, for
// the rows of that beam alone.  A softmax over a union of keys joins from (maximum, sum, weighted values), whoever made the parts.
//
// Bound by the bytes of the keys.  The work is a flat list: a request's block of rows, its key heads, their stages of two pages (128 keys),
// of four with heads of up to 64 numbers. Every block of threads has an even, consecutive share of it, and the copy engine brings its pages
// (128-byte swizzle), ahead across the ends of requests.  Where a share ends inside a block of rows, the sums go out as a partial result; a
// second launch joins those.
//
// 32 heads over 8 of 128 numbers, 16 requests of 8 beams behind 6,000 to 24,000 tokens: 97 us for the 85 that 560 MB take; twice as
// long 166 for 161, of 16 beams 120 for 94, with heads of 64 numbers 60 for 43; 16 heads over 4 of 256 100 for 86, of 16 beams 140
// for 94; one request of 4 beams behind 300 9.1.
#include <math_constants.h>
#include <stdio.h>

#include "tc_common.cuh"

namespace {

typedef __nv_bfloat16 bf16;

constexpr int PAGE = 64;
constexpr int MOST_BEAMS = 32;
constexpr float RESCALE_LOG2 = 8.0f;               // weights may grow to 2^8 before what was summed up is scaled down
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  const bf16* q;
  bf16* out;
  float* part_o;       // [shares][2][rows of a block][hd], not divided by their sums; of a share's first rows (0) and last rows (1)
  float2* part_ml;     // ... maximum (in units of log2), sum
  int2* parts;         // [beams][heads]: first share with a part of the row, number of shares
  const int* table;
  const int* kv_len;
  const int* shared;
  int R, K, nh, nkv, hd, W, n_pages;
  int group;                                       // query heads of a key head
  int row_blocks;                                  // blocks of rows of a request
  int block_rows;                                  // rows of a block
  float scale_log2;
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float low_of(uint32_t two) { return __uint_as_float(two << 16); }
__device__ __forceinline__ float high_of(uint32_t two) { return __uint_as_float(two & 0xffff0000u); }
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bounded wait: false (and *status = code) if the phase did not complete in 4e9 cycles, about two seconds.  Codes are 5, what was waited for
// (1 a place of the ring, 2 keys or values, 3 a stage's description, 4 queries, 5 weights, 6 scores, 7 the products of the stage before, 8 a
// block of rows' sums), and who waited (1 the loads, 2 the products' issuer, 3 the weights and the results).
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

// A block of rows of a request, as a warp knows it; lane b knows beam b.
struct Rows {
  int request, rho0, n_rows;        // rows rho0 .. of the request's beams * group
  int common, head;                 // pages that its beams share; the beam whose table lists them
  int pages;                        // that they read: the shared ones, then each beam's own
  int len, first, own, upto;        // of the lane's beam: keys, first page of its own, pages of its own, of the beams up to it
};

// ... from the lane's beam's length and the request's shared pages, as they stand in memory.
__device__ __forceinline__ Rows rows_of(const Args& a, int block, int len, int shared) {
  const int lane = threadIdx.x & 31, G = a.group;
  Rows x;
  x.request = a.row_blocks == 1 ? block : block / a.row_blocks;
  x.rho0 = (block - x.request * a.row_blocks) * a.block_rows;
  x.n_rows = min(a.block_rows, a.K * G - x.rho0);
  x.len = min(max(len, 0), a.W * PAGE);
  const int most = __reduce_max_sync(0xffffffffu, x.len);
  x.head = __ffs(__ballot_sync(0xffffffffu, lane < a.K && x.len == most)) - 1;
  x.common = min(max(shared, 0), most / PAGE);
  x.first = x.len < x.common * PAGE ? 0 : x.common;        // shorter beams read all they have by themselves
  x.own = lane < a.K && (lane + 1) * G > x.rho0 && lane * G < x.rho0 + x.n_rows ? (x.len - x.first * PAGE + PAGE - 1) / PAGE : 0;
  x.pages = max(1, x.common + __reduce_add_sync(0xffffffffu, x.own));       // (rows without keys have a place as well)
  x.upto = x.own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, x.upto, o);
    if (lane >= o) x.upto += t;
  }
  return x;
}
__device__ __forceinline__ Rows look_up(const Args& a, int block) {
  const int lane = threadIdx.x & 31, request = a.row_blocks == 1 ? block : block / a.row_blocks;
  return rows_of(a, block, lane < a.K ? a.kv_len[request * a.K + lane] : 0, a.shared[request]);
}
// Whether one of two numbers is infinite or none (an exponent of ones carries into the sign's place); the bits say which.  A weight of 0 silences
// neither, so values of pages that not all rows read are looked at: such a value is left out, and that number of the rows that read it becomes no
// number; their other numbers, and other rows, stay what they are.
__device__ __forceinline__ uint32_t not_finite(uint32_t two) { return ((two & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

// Eight values of one key, some of them not finite: those are made 0 and noted for the beams that read the page.  (A call: inlined, what is hardly
// ever done costs the warps registers, 102 us for 97 on the first case, 131 for 119 with 64 rows.)
__device__ __noinline__ void note_values(uint4& place, uint32_t* bad, const unsigned long long* rows, int K, int G, int rho0, int n_rows) {
  uint32_t readers = 0u;
#pragma unroll 1
  for (int b = 0; b < K; ++b) {
    const int row = max(b * G - rho0, 0);
    if (row < min((b + 1) * G - rho0, n_rows)) readers |= (uint32_t)(rows[row / 64] >> (row % 64) & 1ull) << b;
  }
  uint32_t v[4] = {place.x, place.y, place.z, place.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t two = not_finite(v[e]);
    if (two & 0x00008000u) v[e] &= 0xffff0000u, atomicOr(bad + 2 * e, readers);
    if (two & 0x80000000u) v[e] &= 0x0000ffffu, atomicOr(bad + 2 * e + 1, readers);
  }
  place = make_uint4(v[0], v[1], v[2], v[3]);
}

// ---------------------------------------------------------------------------
// The tensor cores of tcgen05, keys on the tile's 128 rows, the beams' queries on its N columns, so that a request's few rows are no padding:
// S' = K Q' and O' = V' P' (two tiles of it for heads of more than 128 numbers), both accumulated in tensor memory.
//   warp 0       walks the block's share of the list and brings keys and values, each to the next place of a ring, by the copy engine
//   warp 1       one lane issues the products; the next stage's scores before this one's values, where its keys are there.  Keys give their place
//                back with the scores, values with their own product
//   warps 4-     two or four groups of four, each with its columns: a thread has one key.  Weights relative to a number a row that is raised
//                only when a score passes it by RESCALE_LOG2 (then the sums and O' are scaled down); P to shared memory, a row a key
// A stage's pages may be different beams' own; a mask of rows goes with each.
//
// With heads of 128 numbers and 32 rows a stage (64 KB) takes 1.3 us, which is memory's rate for a multiprocessor; 3.5 us go by before the first
// copy and 2 more before its scores, 15 between the first share's end and the last one's (multiprocessors are not served alike), 3.5 in the join.
// With heads of 64 numbers the chain of a stage is longer than 32 KB take: a thread has two keys there (78 us by one).  Measured on the first
// case: warp-level products (mma.sync) of the beams' rows padded to 16, 116 us, and 214 for 64 rows, as each of four warps reads all keys from
// shared memory again; two groups of warps for 32 rows 102 for 99.5; lists of single pages, where a share may begin within a stage, 98 for 96,
// and parted beams, whose shares are one stage, 17 for 13 us; keys and values in one place, level, with 64 rows 131 for 122; weights of two
// stages in turn, so that a stage need not wait for the products of the one before, level; keys and values asked for by two pairs of lanes at
// once, level, with 64 rows 130.
// ---------------------------------------------------------------------------
constexpr float NOTHING = -3.402823466e38f;                  // what weights are relative to before a row has seen a key: no number is below

struct Info {                                                // of a stage
  int first, last, final_, whole;                            // of its block of rows' keys in this share; of the share; no mask
  int request, rho0, n_rows, kvh;
  int piece0, piece1;                                        // shares that the block of rows has parts in
  int keys[4];                                               // of its pages, two or four
  unsigned long long rows[4][2];                             // that see the page's keys
};

template <int HDC, int N>
struct Tc {
  static constexpr int HALVES = HDC == 64 && N <= 64 ? 2 : 1;            // of 128 keys, that a thread has one each of
  static constexpr int KEYS = 128 * HALVES, SUB = KEYS / PAGE;           // keys and pages of a stage
  static constexpr int SLABS = HDC / 64, SLAB = KEYS * 128, SLOT = SLABS * SLAB;   // 64 numbers of a stage's keys; its keys, or its values
  static constexpr int TILES = HDC > 128 ? 2 : 1;            // of 128 of the head's numbers in O'
  static constexpr int Q = SLABS * N * 128, P = (N > 64 ? 2 : 1) * KEYS * 128;
  // keys' and values' places, as many as fit beside queries, weights, ref, exchange, descriptions, barriers and notes of values
  static constexpr int infos(int slots) { return slots / 2 + 1; }
  static constexpr int barriers(int slots) { return 2 * slots + infos(slots) + 6; }
  static constexpr int bytes(int slots) {
    return slots * SLOT + Q + P + 4 * N + 16 * N + infos(slots) * (int)sizeof(Info) + barriers(slots) * 8 + 16 + 8 * HDC;
  }
  static constexpr int fit() {
    int slots = 12;
    while (bytes(slots) > 232448) --slots;
    return slots;
  }
  static constexpr int SLOTS = fit(), INFOS = infos(SLOTS);
  static constexpr int AT_Q = SLOTS * SLOT, AT_P = AT_Q + Q, AT_REF = AT_P + P, AT_SWAP = AT_REF + 4 * N, AT_INFO = AT_SWAP + 16 * N,
                       AT_BARS = AT_INFO + INFOS * (int)sizeof(Info), BARS = barriers(SLOTS), AT_BAD = AT_BARS + BARS * 8 + 16, SMEM = AT_BAD + 8 * HDC;
  static constexpr int AT_O = 2 * HALVES * N, COLS_USED = AT_O + TILES * N;     // of tensor memory: two S', O'
  static constexpr int COLS = COLS_USED <= 64 ? 64 : COLS_USED <= 128 ? 128 : COLS_USED <= 256 ? 256 : 512;
  static_assert(COLS_USED <= 512, "tensor memory");
  static constexpr int GROUPS = N > 16 ? 4 : 2, HALF = N / GROUPS;      // groups of four warps, columns of each
  static constexpr int PLACES = 1024;                                   // of the list, whose stages are counted
  static constexpr int WARPS = 4 * GROUPS, THREADS = 128 + 32 * WARPS;
  static_assert(SLOTS >= 2 && SMEM == bytes(SLOTS) && SMEM <= 232448, "shared memory of a block");
  static __device__ __forceinline__ int stages_of(const Rows& x) { return (x.pages + SUB - 1) / SUB; }
};

// Where a ring's next stage stands: keys take a place, values the next one.
template <int SLOTS>
struct Ring {
  int at;
  uint32_t phase = 0;
  __device__ __forceinline__ explicit Ring(int first) : at(first) {}
  __device__ __forceinline__ void step(int by) {
    at += by;
    if (at >= SLOTS) at -= SLOTS, phase ^= 1;
  }
};

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0u;
}
__device__ __forceinline__ float warp_top(float v) {                 // the largest of a warp's numbers (one that is none is passed over)
  float top;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(v));
  return top;
}
__device__ __forceinline__ bool elected() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0u;
}
// A barrier of a group of four warps that tells all whether any of its threads says `yes`.
__device__ __forceinline__ bool group_any(int barrier, bool yes) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(barrier), "r"((uint32_t)yes)
      : "memory");
  return any != 0u;
}
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr, uint32_t lead, uint32_t stride) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)((lead >> 4) & 0x3FFF) << 16 | (uint64_t)((stride >> 4) & 0x3FFF) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "f"(r[0]), "f"(r[1]), "f"(r[2]),
               "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Rows [from, to) of a block, as bits.
__device__ __forceinline__ void add_rows(unsigned long long (&bits)[2], int from, int to) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int a = min(max(from - 64 * w, 0), 64), b = min(max(to - 64 * w, 0), 64);
    if (b > a) bits[w] |= (b - a == 64 ? ~0ull : ((1ull << (b - a)) - 1ull)) << a;
  }
}

// out[c] = the sum of v[c] over the warp's lanes, for C columns (8, 16 or 32).
template <int C>
__device__ __forceinline__ void columns_summed(const float (&v)[C], float* out) {
  const int lane = threadIdx.x & 31;
  float t[C];
#pragma unroll
  for (int c = 0; c < C; ++c) t[c] = v[c];
  int o = 16, left = C;
#pragma unroll
  for (int step = 0; step < 5; ++step, o >>= 1) {
    if (left > 1) {
      left >>= 1;
      const bool up = (lane & o) != 0;
#pragma unroll
      for (int c = 0; c < C / 2; ++c) {
        if (c < left) {
          const float mine = up ? t[left + c] : t[c], other = up ? t[c] : t[left + c];
          t[c] = mine + __shfl_xor_sync(0xffffffffu, other, o);
        }
      }
    } else {
      t[0] += __shfl_xor_sync(0xffffffffu, t[0], o);
    }
  }
  // lane bits from the top name the column, as far as they were needed
  constexpr int BITS = C == 8 ? 3 : C == 16 ? 4 : 5;
  if ((lane & ((1 << (5 - BITS)) - 1)) == 0) out[lane >> (5 - BITS)] = t[0];
}

template <int HDC, int N>
__global__ void __launch_bounds__(Tc<HDC, N>::THREADS, 1) beam_attention_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                        const __grid_constant__ CUtensorMap map_v, const Args a,
                                                                        int* __restrict__ status) {
  typedef Tc<HDC, N> C;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, G = a.group, hd = a.hd;
  const uint32_t base = jb::smem_u32(smem), q_at = base + C::AT_Q, p_at = base + C::AT_P;
  float* ref = reinterpret_cast<float*>(smem + C::AT_REF);             // [N] in units of log2
  float* swap = reinterpret_cast<float*>(smem + C::AT_SWAP);           // [4][N]
  Info* info = reinterpret_cast<Info*>(smem + C::AT_INFO);             // [INFOS]
  const uint32_t full = base + C::AT_BARS, empty = full + 8 * C::SLOTS, told = empty + 8 * C::SLOTS, s_full = told + 8 * C::INFOS, p_full = s_full + 16,
                 pv_done = p_full + 8, q_full = pv_done + 8, o_full = q_full + 8;
  // [block of rows' parity][number of the head]: beams that read a value there that is not finite, as the group that looks there has found
  uint32_t (*bad)[HDC] = reinterpret_cast<uint32_t (*)[HDC]>(smem + C::AT_BAD);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + C::AT_BARS + C::BARS * 8);
  if (tid == 0) {
    for (int i = 0; i < C::SLOTS; ++i) jb::mbar_init(full + 8 * i, 1), jb::mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < C::INFOS; ++i) jb::mbar_init(told + 8 * i, 1);
    jb::mbar_init(s_full, 1), jb::mbar_init(s_full + 8, 1), jb::mbar_init(p_full, C::WARPS), jb::mbar_init(pv_done, 1), jb::mbar_init(q_full, C::WARPS);
    jb::mbar_init(o_full, 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) jb::tmem_alloc<C::COLS>(jb::smem_u32((const void*)tmem_slot));
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  // ---- the list's length: every warp has some of its places, several requests' lengths on their way at a time ----
  int* sums = reinterpret_cast<int*>(smem + C::AT_P);                  // [places] (P is not there yet)
  const int blocks = a.R * a.row_blocks, chunk = (blocks + C::PLACES - 1) / C::PLACES, places = (blocks + chunk - 1) / chunk;
  constexpr int AHEAD = 4;
  for (int p0 = warp; p0 < places; p0 += C::THREADS / 32 * AHEAD) {
    int stages[AHEAD] = {};
    for (int i = 0; i < chunk; ++i) {
      int len[AHEAD], shared[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int block = min((p0 + u * (C::THREADS / 32)) * chunk + i, blocks - 1), request = a.row_blocks == 1 ? block : block / a.row_blocks;
        len[u] = lane < a.K ? a.kv_len[request * a.K + lane] : 0, shared[u] = a.shared[request];
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int block = (p0 + u * (C::THREADS / 32)) * chunk + i;
        if (block < blocks) stages[u] += C::stages_of(rows_of(a, block, len[u], shared[u]));
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (lane == 0 && p0 + u * (C::THREADS / 32) < places) sums[p0 + u * (C::THREADS / 32)] = stages[u] * a.nkv;
  }
  jb::tc_fence_before();
  __syncthreads();
  jb::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (warp == 0) {
    const int each = (places + 31) / 32;
    int mine = 0;
    for (int i = lane * each; i < min(lane * each + each, places); ++i) mine += sums[i];
    int up = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += t;
    }
    const int total = __shfl_sync(0xffffffffu, up, 31);
    const int per = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);     // (a short list: no share with parts of two blocks of rows)
    const int begin = min((int)blockIdx.x * per, total), end = min(begin + per, total);
    const int owner = begin < end ? __ffs(__ballot_sync(0xffffffffu, begin < up)) - 1 : 0, before_owner = __shfl_sync(0xffffffffu, up - mine, owner);
    int block = 0, kvh = 0, turn = 0, stages = 1, at = begin;
    Ring<C::SLOTS> slot(0);
    Ring<C::INFOS> note(0);
    bool ok = true;
    Rows x{};
    if (begin >= end) {                                                // nothing: one stage that says so
      if (lane == 0) {
        info[0].final_ = 2;
        jb::mbar_arrive(told);
        jb::mbar_arrive(full);
      }
    } else {
      int before = before_owner, t = owner * each;
      while (begin >= before + sums[t]) before += sums[t++];
      for (block = t * chunk;; ++block) {
        x = look_up(a, block);
        stages = C::stages_of(x);
        if (begin < before + stages * a.nkv) break;
        before += stages * a.nkv;
      }
      kvh = (begin - before) / stages;
      turn = begin - before - kvh * stages;
    }
    unsigned long long joining[2] = {0ull, 0ull}, all[2] = {0ull, 0ull};
    int piece0 = 0, piece1 = 0;
    auto entered = [&]() {                                             // rows that read the shared pages; all rows
      joining[0] = joining[1] = all[0] = all[1] = 0ull;
      add_rows(all, 0, x.n_rows);
      const unsigned beams = a.K == 32 ? ~0u : (1u << a.K) - 1u;
      unsigned who = __ballot_sync(0xffffffffu, lane < a.K && x.len >= x.common * PAGE);
      if (who == beams) {
        joining[0] = all[0], joining[1] = all[1];
        return;
      }
      while (who) {
        const int b = __ffs(who) - 1;
        who &= who - 1;
        add_rows(joining, max(b * G - x.rho0, 0), min((b + 1) * G - x.rho0, x.n_rows));
      }
    };
    auto begun = [&]() {                                               // the shares that this head's pages lie in
      piece0 = (at - turn) / per, piece1 = (at - turn + stages - 1) / per;
    };
    // The lanes look up 32 pages at a time; of a stage's, lanes 0 and 1 have one each.
    int ahead = 0, keys = 0, beam = -1, page = -1;                     // the first one's place; the lane's: keys, beam (-1: all that share it), page
    auto find = [&]() {
      ahead = turn * C::SUB;
      beam = -1, keys = 0, page = -1;
      const int mine = ahead + lane, j = mine - x.common;
      const bool there = mine < x.pages && at + lane / C::SUB < end;
      const int* entry = nullptr;
      if (there && j < 0) {
        keys = PAGE;
        entry = a.table + ((size_t)x.request * a.K + x.head) * a.W + mine;
      }
      if (ahead + 31 >= x.common) {                                    // beams' own
        int b = 0;
        for (int k = 0; k < a.K; ++k) b += __shfl_sync(0xffffffffu, x.upto, k) <= j;
        const int who = min(b, 31), first = __shfl_sync(0xffffffffu, x.first, who), before = __shfl_sync(0xffffffffu, x.upto - x.own, who),
                  len = __shfl_sync(0xffffffffu, x.len, who);
        if (there && j >= 0 && b < a.K) {                              // (rows without keys: nobody's)
          const int column = first + j - before;
          beam = b, keys = min(PAGE, len - column * PAGE);
          entry = a.table + ((size_t)x.request * a.K + b) * a.W + column;
        }
      }
      if (entry != nullptr) page = *entry;
    };
    if (at < end) {
      find();                                                          // (the rest while the pages' numbers are on their way)
      entered();
      begun();
    }
    while (at < end) {
      if (turn * C::SUB >= ahead + 32) find();
      const int n = min(C::SUB, x.pages - turn * C::SUB), from = turn * C::SUB - ahead + (lane & (C::SUB - 1));
      const int keys0 = __shfl_sync(0xffffffffu, keys, from), beam0 = __shfl_sync(0xffffffffu, beam, from), page0 = __shfl_sync(0xffffffffu, page, from);
      unsigned long long rows[2] = {joining[0], joining[1]};
      if (beam0 >= 0) {
        rows[0] = rows[1] = 0ull;
        add_rows(rows, max(beam0 * G - x.rho0, 0), min((beam0 + 1) * G - x.rho0, x.n_rows));
      }
      const bool there = lane < n && keys0 > 0 && page0 >= 0 && page0 < a.n_pages;    // (no page: no keys)
      const unsigned loads = __ballot_sync(0xffffffffu, there);
      const bool whole = __all_sync(0xffffffffu, lane >= C::SUB || (there && keys0 == PAGE && rows[0] == all[0] && rows[1] == all[1]));
      ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * slot.at, slot.phase ^ 1, status, 511));
      if (!ok) break;
      Info& to = info[note.at];
      if (lane < C::SUB) to.keys[lane] = there ? keys0 : 0, to.rows[lane][0] = rows[0], to.rows[lane][1] = rows[1];
      if (lane == 0) {
        to.first = at == begin || turn == 0, to.last = turn + 1 == stages || at + 1 == end, to.final_ = at + 1 == end, to.whole = whole;
        to.request = x.request, to.rho0 = x.rho0, to.n_rows = x.n_rows, to.kvh = kvh;
        to.piece0 = piece0, to.piece1 = piece1;
      }
      __syncwarp();
      if (lane == 0) jb::mbar_arrive(told + 8 * note.at);
      note.step(1);
      const int row = (page0 * a.nkv + kvh) * PAGE;
#pragma unroll
      for (int half = 0; half < 2; ++half) {                           // keys, values
        if (half > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * slot.at, slot.phase ^ 1, status, 511));
          if (!ok) break;
        }
        const uint32_t here = full + 8 * slot.at, place = base + slot.at * C::SLOT + lane * PAGE * 128;
        if (lane == 0) {
          if (loads) jb::mbar_expect_tx(here, __popc(loads) * C::SLABS * PAGE * 128);
          else jb::mbar_arrive(here);
        }
        __syncwarp();
        if (there) {
#pragma unroll
          for (int h = 0; h < C::SLABS; ++h) jb::tma_load_2d(place + h * C::SLAB, half ? &map_v : &map_k, here, h * 64, row);
        }
        slot.step(1);
      }
      if (!ok) break;
      ++at, ++turn;
      if (at < end && turn == stages) {
        turn = 0;
        const bool enters = ++kvh == a.nkv;
        if (enters) kvh = 0, x = look_up(a, ++block), stages = C::stages_of(x);
        find();
        if (enters) entered();
        begun();
      }
    }
    // gave up: what is still on its way arrives before the block ends (or its wait gives up as well)
    if (!ok && lane == 0)
      for (int i = 0; i < C::SLOTS; ++i) mbar_wait(full + 8 * i, i < slot.at ? slot.phase : slot.phase ^ 1, status, 521);
  } else if (warp == 1) {
    if (elected()) {
      const uint32_t idesc_s = jb::instr_desc_bf16(N), idesc_o = jb::instr_desc_bf16(N) | (1u << 15) | (1u << 16);   // values and weights: MN-major
      const uint32_t o_col = tmem + C::AT_O;
      const uint64_t p = desc_mn_sw128(p_at, C::KEYS * 128, 1024);
      Ring<C::SLOTS> ks(0), vs(1);
      Ring<C::INFOS> note(0);
      int it = 0, turn = 0;
      bool ok = true, ahead = false;                                   // the stage's scores are under way already
      auto scores = [&](int buffer) {
        const uint32_t k_s = base + ks.at * C::SLOT;
        jb::tc_fence_after();
#pragma unroll
        for (int t = 0; t < C::HALVES; ++t)
#pragma unroll
          for (int h = 0; h < C::SLABS; ++h) {
            const uint64_t k = jb::smem_desc_sw128(k_s + h * C::SLAB + t * 128 * 128), q = jb::smem_desc_sw128(q_at + h * N * 128);
#pragma unroll
            for (int i = 0; i < 4; ++i) jb::umma_bf16(tmem + (buffer * C::HALVES + t) * N, k + 2 * i, q + 2 * i, idesc_s, (h | i) ? 1u : 0u);
          }
        jb::umma_commit(s_full + 8 * buffer);
        jb::umma_commit(empty + 8 * ks.at);
        ks.step(2);
      };
      for (;; ++it) {
        const Info& x = info[note.at];
        if (!ahead) {
          ok = mbar_wait(full + 8 * ks.at, ks.phase, status, 522) && mbar_wait(told + 8 * note.at, note.phase, status, 532);
          if (!ok || x.final_ == 2) break;
          if (x.first) ok = mbar_wait(q_full, turn++ & 1, status, 542);
          if (!ok) break;
          scores(it & 1);
        }
        const bool first = x.first, last = x.last, final_ = x.final_;
        ahead = false;
        if (!last && mbar_test(full + 8 * ks.at, ks.phase)) {
          scores((it + 1) & 1);
          ahead = true;
        }
        ok = mbar_wait(full + 8 * vs.at, vs.phase, status, 522) && mbar_wait(p_full, it & 1, status, 552);
        if (!ok) break;
        jb::tc_fence_after();
        const uint64_t v = desc_mn_sw128(base + vs.at * C::SLOT, C::SLAB, 1024);         // (further on by 16 bytes a unit)
#pragma unroll
        for (int m = 0; m < C::TILES; ++m)
#pragma unroll
          for (int i = 0; i < C::KEYS / 16; ++i)
            jb::umma_bf16(o_col + m * N, v + (m * 2 * C::SLAB + i * 2048) / 16, p + i * 2048 / 16, idesc_o, first && i == 0 ? 0u : 1u);
        jb::umma_commit(pv_done);
        jb::umma_commit(empty + 8 * vs.at);
        if (last) jb::umma_commit(o_full), jb::mbar_arrive(o_full);    // (by itself as well: what the groups wrote before is seen behind it)
        if (final_) break;
        vs.step(2);
        note.step(1);
      }
    }
  } else if (warp >= 4) {
    const int group = (warp - 4) >> 2, quarter = warp & 3, key = quarter * 32 + lane, c0 = group * C::HALF;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    float* my_ref = ref + c0;
    float l[C::HALF];
    Ring<C::SLOTS> vs(1);
    Ring<C::INFOS> note(0);
    int turn = 0, request = 0, rho0 = 0, n_rows = 0, kvh = 0;
    bool ok = true, first = true;
    for (int it = 0;; ++it) {
      // a block of rows begins: its queries, by all groups, while its first keys are on their way
      const Info* x = info + note.at;
      ok = ok && mbar_wait(told + 8 * note.at, note.phase, status, 533);
      if (first) {
        if (group_any(1 + group, !ok)) break;                          // (a wait ran out, of one of the group's warps: all leave)
        request = x->request, rho0 = x->rho0, n_rows = x->n_rows, kvh = x->kvh;
        if (x->final_ == 2) break;                                     // (the block has no share)
        for (int ch = tid - 128; ch < N * C::SLABS * 8; ch += 32 * C::WARPS) {
          const int row = ch / (C::SLABS * 8), piece = ch % (C::SLABS * 8), rho = rho0 + row;
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (row < n_rows && piece * 8 < hd)
            v = *reinterpret_cast<const uint4*>(a.q + (((size_t)request * a.K + rho / G) * a.nh + kvh * G + rho % G) * hd + piece * 8);
          *reinterpret_cast<uint4*>(smem + C::AT_Q + (piece / 8) * N * 128 + row * 128 + (((piece % 8) ^ (row & 7)) << 4)) = v;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) jb::mbar_arrive(q_full);
        if (key < C::HALF) my_ref[key] = NOTHING;
        for (int d = key; d < HDC; d += 128)
          if (d / 8 % C::GROUPS == group) bad[turn & 1][d] = 0u;
#pragma unroll
        for (int c = 0; c < C::HALF; ++c) l[c] = 0.0f;
      }
      if (group_any(1 + group, !ok)) break;
      const bool last = x->last;
      const int final_ = x->final_, in_page = (quarter & 1) * 32 + lane;
      const bool masked = !x->whole;
      unsigned long long rows[C::HALVES] = {};
      if (masked) {
        // values behind the last key, or that are no finite numbers: a weight of 0 does not silence them (a part of the head's numbers a
        // group; while the scores are made)
        ok = ok && mbar_wait(full + 8 * vs.at, vs.phase, status, 523);
#pragma unroll
        for (int t = 0; t < C::HALVES; ++t) {
          const int sub = t * 2 + (quarter >> 1);
          const bool behind = in_page >= x->keys[sub];
          rows[t] = behind ? 0ull : x->rows[sub][c0 / 64] >> (c0 % 64);
          uint8_t* values = smem + vs.at * C::SLOT + (t * 128 + key) * 128;
          uint32_t odd = 0u;
#pragma unroll
          for (int p = 0; p < C::SLABS * 8 / C::GROUPS; ++p) {
            const int at = p * C::GROUPS + group;
            const uint4 v = *reinterpret_cast<const uint4*>(values + (at / 8) * C::SLAB + (((at ^ key) & 7) << 4));
            odd |= not_finite(v.x) | not_finite(v.y) | not_finite(v.z) | not_finite(v.w);
          }
          if (odd != 0u || behind) {
#pragma unroll 1
            for (int at = group; at < C::SLABS * 8; at += C::GROUPS) {
              uint4* place = reinterpret_cast<uint4*>(values + (at / 8) * C::SLAB + (((at ^ key) & 7) << 4));
              if (odd != 0u && !behind) note_values(*place, bad[turn & 1] + at * 8, x->rows[sub], a.K, G, rho0, n_rows);
              else *place = make_uint4(0u, 0u, 0u, 0u);
            }
          }
        }
      }
      ok = ok && mbar_wait(s_full + 8 * (it & 1), (it >> 1) & 1, status, 563);
      jb::tc_fence_after();
      bool rest = it == 0;                                             // P is free, and O' at rest
      auto settle = [&]() {
        if (!rest) ok = ok && mbar_wait(pv_done, (it - 1) & 1, status, 573), jb::tc_fence_after();
        rest = true;
      };
      float s[C::HALVES][C::HALF];
      auto scores = [&]() {
#pragma unroll
        for (int t = 0; t < C::HALVES; ++t)
#pragma unroll
          for (int c = 0; c < C::HALF; c += 8) {
            float v[8];
            jb::tmem_ld8(lanes + ((it & 1) * C::HALVES + t) * N + c0 + c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[t][c + e] = v[e];
          }
        jb::tmem_ld_wait();
        // (rounded by itself: a fused product less the row's number, which is rounded, would leave 2^-24 of a large score as a power)
#pragma unroll
        for (int t = 0; t < C::HALVES; ++t)
#pragma unroll
          for (int c = 0; c < C::HALF; ++c) s[t][c] = __fmul_rn(s[t][c], a.scale_log2);
        if (masked) {
#pragma unroll
          for (int t = 0; t < C::HALVES; ++t)
#pragma unroll
            for (int c = 0; c < C::HALF; ++c)
              if (!((rows[t] >> c) & 1ull)) s[t][c] = -CUDART_INF_F;
        }
      };
      scores();
      // powers relative to the rows' numbers
      float high = -CUDART_INF_F;
#pragma unroll
      for (int c = 0; c < C::HALF; c += 4) {
        const float4 r = *reinterpret_cast<const float4*>(my_ref + c);
#pragma unroll
        for (int t = 0; t < C::HALVES; ++t) {
          float* y = s[t] + c;
          y[0] -= r.x, y[1] -= r.y, y[2] -= r.z, y[3] -= r.w;
          high = fmaxf(high, fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
        }
      }
      if (group_any(1 + group, high > RESCALE_LOG2)) {
        // the rows' largest over the block's keys
        settle();
        scores();
#pragma unroll
        for (int c = 0; c < C::HALF; ++c) {
          float most = s[0][c];
#pragma unroll
          for (int t = 1; t < C::HALVES; ++t) most = fmaxf(most, s[t][c]);
          const float top = warp_top(most);
          if (lane == 0) swap[quarter * N + c0 + c] = top;
        }
        group_any(1 + group, false);
        float old = 0.0f, now = 0.0f;
        if (key < C::HALF) {
          const float* t = swap + c0 + key;
          old = my_ref[key];
          now = fmaxf(old, fmaxf(fmaxf(t[0], t[N]), fmaxf(t[2 * N], t[3 * N])));
        }
        group_any(1 + group, false);
        if (key < C::HALF) my_ref[key] = now, swap[c0 + key] = fast_exp2(old - now);
        group_any(1 + group, false);
#pragma unroll
        for (int c = 0; c < C::HALF; c += 8) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
#pragma unroll
            for (int t = 0; t < C::HALVES; ++t) s[t][c + e] -= my_ref[c + e];
            f[e] = swap[c0 + c + e], l[c + e] *= f[e];
          }
          if (!first) {
#pragma unroll
            for (int m = 0; m < C::TILES; ++m) {
              float v[8];
              jb::tmem_ld8(lanes + C::AT_O + m * N + c0 + c, v);
              jb::tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] *= f[e];
              tmem_st8(lanes + C::AT_O + m * N + c0 + c, v);
            }
          }
        }
        tmem_st_wait();
      }
      uint32_t w[C::HALVES][C::HALF / 2];
#pragma unroll
      for (int t = 0; t < C::HALVES; ++t)
#pragma unroll
        for (int c = 0; c < C::HALF; c += 2) {
          const uint32_t two = pack_bf16(fast_exp2(s[t][c]), fast_exp2(s[t][c + 1]));
          l[c] += low_of(two), l[c + 1] += high_of(two);               // (as they are rounded: a weight that outdoes all others costs nothing)
          w[t][c / 2] = two;
        }
      settle();
#pragma unroll
      for (int t = 0; t < C::HALVES; ++t) {
        uint8_t* p_row = smem + C::AT_P + (c0 / 64) * C::KEYS * 128 + (t * 128 + key) * 128;
#pragma unroll
        for (int c = 0; c < C::HALF; c += 8) {
          const int piece = (c0 % 64 + c) / 8;
          *reinterpret_cast<uint4*>(p_row + ((piece ^ (key & 7)) << 4)) =
              make_uint4(w[t][c / 2], w[t][c / 2 + 1], w[t][c / 2 + 2], w[t][c / 2 + 3]);
        }
      }
      const int piece0 = x->piece0, piece1 = x->piece1;                // (read before the stage is given back)
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      jb::tc_fence_before();
      __syncwarp();
      if (lane == 0) jb::mbar_arrive(p_full);
      if (last) {
        group_any(1 + group, false);                                   // (nobody reads there any longer)
        // the sums over the keys: half the columns go to the other half of the lanes, and so on, until a lane has one
        columns_summed<C::HALF>(l, swap + quarter * N + c0);
        const int spoil = turn & 1;
        ok = ok && mbar_wait(o_full, turn++ & 1, status, 583);
        jb::tc_fence_after();
        group_any(1 + group, false);
        const int piece = (int)blockIdx.x;
        const bool complete = piece0 == piece1;
        const size_t record = ((size_t)piece * 2 + (piece == piece0 ? 1 : 0)) * N;
        // a thread a row: where its numbers go (times the heads' numbers), and what they are divided by
        if (key < C::HALF) {
          const int row = c0 + key, rho = rho0 + row;
          float* t = swap + c0 + key;
          const float sum = (t[0] + t[N]) + (t[2 * N] + t[3 * N]);
          t[0] = complete ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
          if (row < n_rows) {
            const int item = (request * a.K + rho / G) * a.nh + kvh * G + rho % G;
            t[N] = __int_as_float(complete ? item : (int)record + row);
            if (piece == piece0) a.parts[item] = make_int2(piece0, piece1 - piece0 + 1);
            if (!complete) a.part_ml[record + row] = make_float2(sum != sum ? 0.0f : sum == 0.0f ? -CUDART_INF_F : my_ref[key], sum);
          }
        }
        group_any(1 + group, false);
#pragma unroll
        for (int c = 0; c < C::HALF; c += 8) {
#pragma unroll
          for (int m = 0; m < C::TILES; ++m) {
            float v[8];
            jb::tmem_ld8(lanes + C::AT_O + m * N + c0 + c, v);
            jb::tmem_ld_wait();
            if (key + 128 * m < hd) {
              const uint32_t spoilt = bad[spoil][key + 128 * m];
              if (spoilt != 0u) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (spoilt >> ((rho0 + c0 + c + e) / G & 31) & 1u) v[e] = CUDART_NAN_F;
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int row = c0 + c + e;
                if (row < n_rows) {
                  const size_t to = (size_t)__float_as_int(swap[N + row]) * hd + key + 128 * m;
                  if (complete) a.out[to] = __float2bfloat16_rn(v[e] * swap[row]);
                  else a.part_o[to] = v[e];
                }
              }
            }
          }
        }
        jb::tc_fence_before();
        group_any(1 + group, false);                                   // (what was exchanged has been read)
      }
      first = last;
      if (final_) break;
      vs.step(2);
      note.step(1);
    }
  }
  jb::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    jb::tc_fence_after();
    jb::tmem_dealloc<C::COLS>(tmem);
  }
}

// The parts of a (beam, head)'s keys joined, where there are several, by PER warps, each of which takes every PER-th, several on their way at
// a time.
constexpr int JOIN_WARPS = 4;
template <int PER>
__global__ void __launch_bounds__(32 * JOIN_WARPS) beam_attention_join_kernel(const Args a, int rows, int shares) {
  __shared__ float4 sums[PER > 1 ? PER : 1][PER > 1 ? 64 : 1];
  __shared__ float2 ml_of[PER];
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  const int item = blockIdx.x * (JOIN_WARPS / PER) + (threadIdx.x >> 5) / PER, warp = (threadIdx.x >> 5) % PER, lane = threadIdx.x & 31;
  const int G = a.nh / a.nkv;
  if (item >= a.R * a.K * a.nh) return;
  const int2 parts = a.parts[item];
  if (parts.y <= 1 || parts.x < 0 || parts.y > shares - parts.x) return;    // (what a launch whose wait ran out has left is not followed)
  const int head = item % a.nh, beam = item / a.nh % a.K, row = (beam * G + head % G) % rows;
  auto record = [&](int p) { return ((size_t)(parts.x + p) * 2 + (p == 0 ? 1 : 0)) * rows + row; };
  constexpr int AHEAD = 4;
  float4 o[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
  float most = -CUDART_INF_F, sum = 0.0f;
  for (int p0 = warp; p0 < parts.y; p0 += PER * AHEAD) {
    float2 ml[AHEAD];
    float4 v[AHEAD][2];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int p = p0 + u * PER;
      ml[u] = make_float2(-CUDART_INF_F, 0.0f);
      v[u][0] = v[u][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (p < parts.y) {
        const float* from = a.part_o + record(p) * a.hd;
        ml[u] = a.part_ml[record(p)];
        if (lane * 4 < a.hd) v[u][0] = *reinterpret_cast<const float4*>(from + lane * 4);
        if (lane * 4 + 128 < a.hd) v[u][1] = *reinterpret_cast<const float4*>(from + lane * 4 + 128);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const float top = fmaxf(most, ml[u].x);
      if (top == -CUDART_INF_F) continue;
      const float f = fast_exp2(most - top), g = fast_exp2(ml[u].x - top);
      most = top;
      sum = fmaf(sum, f, g * ml[u].y);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        o[h].x = fmaf(o[h].x, f, g * v[u][h].x), o[h].y = fmaf(o[h].y, f, g * v[u][h].y);
        o[h].z = fmaf(o[h].z, f, g * v[u][h].z), o[h].w = fmaf(o[h].w, f, g * v[u][h].w);
      }
    }
  }
  if constexpr (PER == 1) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (lane * 4 + 128 * h < a.hd)
        *reinterpret_cast<uint2*>(a.out + (size_t)item * a.hd + lane * 4 + 128 * h) =
            make_uint2(pack_bf16(o[h].x * inv, o[h].y * inv), pack_bf16(o[h].z * inv, o[h].w * inv));
  } else {
    static_assert(PER == JOIN_WARPS, "a block's barrier");
    if (lane == 0) ml_of[warp] = make_float2(most, sum);
    sums[warp][lane] = o[0], sums[warp][32 + lane] = o[1];
    __syncthreads();
    float top = -CUDART_INF_F, all = 0.0f;
#pragma unroll
    for (int w = 0; w < PER; ++w) top = fmaxf(top, ml_of[w].x);
    const float use = top == -CUDART_INF_F ? 0.0f : top;
    float f[PER];
#pragma unroll
    for (int w = 0; w < PER; ++w) f[w] = fast_exp2(ml_of[w].x - use), all = fmaf(f[w], ml_of[w].y, all);
    const float inv = all == 0.0f ? 0.0f : 1.0f / all;
    for (int d = threadIdx.x; d < a.hd; d += 32 * JOIN_WARPS) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < PER; ++w) t = fmaf(f[w], reinterpret_cast<const float*>(sums[w])[d], t);
      a.out[(size_t)item * a.hd + d] = __float2bfloat16_rn(t * inv);
    }
  }
}

// The kernel's shared memory, asked for once a device.
template <typename Kernel>
cudaError_t allow(Kernel kernel, int bytes, bool (&ready)[64]) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess || (device < 64 && ready[device])) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && device < 64) ready[device] = true;
  return e;
}
// `shares`: of the list, how many.  A block of rows that is cut into many parts has a block of warps a row, others a warp.  Both sides over 180
// shapes (4 and 8 beams of 1 to 64 requests, three kinds of heads, 300 to 16,000 tokens), by shares a block of rows: at 0.3 53 us by a warp and 66
// by a block, at 2.3 13.9 and 15.0, at 4.6 level, at 9 32 and 30, at 18 16.2 and 13.7, at 37 27.5 and 20.3.  From 4 on costs 0.9 % on average, 15 %
// at most (from 6 or 8 on 0.5 %).
cudaError_t join(const Args& a, int rows, int shares, cudaStream_t stream) {
  const int items = a.R * a.K * a.nh;
  if (shares > 4 * a.R * a.row_blocks * a.nkv) {
    jb::Launch cfg(dim3(items), dim3(32 * JOIN_WARPS), 0, stream);
    return cudaLaunchKernelEx(&cfg.c, beam_attention_join_kernel<JOIN_WARPS>, a, rows, shares);
  }
  jb::Launch cfg(dim3((items + JOIN_WARPS - 1) / JOIN_WARPS), dim3(32 * JOIN_WARPS), 0, stream);
  return cudaLaunchKernelEx(&cfg.c, beam_attention_join_kernel<1>, a, rows, shares);
}
template <int HDC, int N>
cudaError_t tc_go(const CUtensorMap* maps, Args a, int blocks, int* status, cudaStream_t stream) {
  typedef Tc<HDC, N> C;
  static bool ready[64] = {};
  cudaError_t e = allow(beam_attention_kernel<HDC, N>, C::SMEM, ready);
  if (e != cudaSuccess) return e;
  jb::Launch cfg(dim3(blocks), dim3(C::THREADS), C::SMEM, stream);
  e = cudaLaunchKernelEx(&cfg.c, beam_attention_kernel<HDC, N>, maps[0], maps[1], a, status);
  return e != cudaSuccess ? e : join(a, N, blocks, stream);
}
template <int HDC>
cudaError_t tc_for(const CUtensorMap* maps, const Args& a, int blocks, int* status, cudaStream_t stream) {
  if (a.block_rows == 16) return tc_go<HDC, 16>(maps, a, blocks, status, stream);
  if (a.block_rows == 32) return tc_go<HDC, 32>(maps, a, blocks, status, stream);
  if constexpr (HDC <= 128)
    if (a.block_rows == 128) return tc_go<HDC, 128>(maps, a, blocks, status, stream);
  return tc_go<HDC, 64>(maps, a, blocks, status, stream);
}

}  // namespace

// part: float32 scratch of 2 * blocks * rows * (hd + 2) + 2 R K nh numbers.  rows: of a block, 16, 32, 64 or (heads of up to 128 numbers) 128.
JB_EXPORT int jb_attention_beams(const void* q, const void* k_cache, const void* v_cache, void* out, void* part, const int* table,
                                 const int* kv_len, const int* shared, int R, int K, int nh, int nkv, int hd, int W, int n_pages, int blocks,
                                 int rows, float scale, int* status, cudaStream_t stream) {
  JB_REFUSE(R < 1 || K < 1 || K > MOST_BEAMS || nkv < 1 || nh < nkv || nh % nkv || hd < 8 || hd > 256 || hd % 8 || W < 1 || W > 0x7fffffff / PAGE ||
                n_pages < 1 || (long long)R * K * nh > 0x7fffffffLL || (long long)n_pages * nkv * PAGE > 0x7fffffffLL || blocks < 1 || !(scale > 0.0f),
            "attention_beams: %d groups of %d beams, %d heads over %d of %d numbers, %d pages a row of %d, %d blocks, scale %g", R, K, nh, nkv, hd,
            W, n_pages, blocks, scale);
  JB_REFUSE(rows != 16 && rows != 32 && rows != 64 && (rows != 128 || hd > 128), "attention_beams: blocks of %d rows", rows);
  JB_REFUSE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)part) % 16, "attention_beams: q, out or workspace not on a boundary of 16 bytes");
  const size_t row_bytes = (size_t)R * K * nh * hd * 2, cache_bytes = (size_t)n_pages * nkv * PAGE * hd * 2;
  auto over = [&](const void* other, size_t bytes) { return (uintptr_t)out < (uintptr_t)other + bytes && (uintptr_t)other < (uintptr_t)out + row_bytes; };
  if (over(q, row_bytes) || over(k_cache, cache_bytes) || over(v_cache, cache_bytes) || over(table, (size_t)R * K * W * 4) ||
      over(kv_len, (size_t)R * K * 4) || over(shared, (size_t)R * 4))
    return JB_ERR_OVERLAP;
  CUtensorMap maps[2];
  if (!jb::make_map_64(&maps[0], k_cache, (uint64_t)n_pages * nkv * PAGE, hd, PAGE, true) ||
      !jb::make_map_64(&maps[1], v_cache, (uint64_t)n_pages * nkv * PAGE, hd, PAGE, true))
    return JB_ERR_TENSORMAP;
  Args a{};
  a.q = (const bf16*)q, a.out = (bf16*)out, a.table = table, a.kv_len = kv_len, a.shared = shared;
  const size_t records = (size_t)blocks * 2 * rows;
  a.part_o = (float*)part, a.part_ml = (float2*)(a.part_o + records * hd), a.parts = (int2*)(a.part_ml + records);
  a.R = R, a.K = K, a.nh = nh, a.nkv = nkv, a.hd = hd, a.W = W, a.n_pages = n_pages;
  a.group = nh / nkv, a.scale_log2 = scale * LOG2E, a.block_rows = rows;
  a.row_blocks = (K * (nh / nkv) + rows - 1) / rows;
  return (int)(hd > 128 ? tc_for<256>(maps, a, blocks, status, stream) : hd > 64 ? tc_for<128>(maps, a, blocks, status, stream)
                                                                                : tc_for<64>(maps, a, blocks, status, stream));
}
