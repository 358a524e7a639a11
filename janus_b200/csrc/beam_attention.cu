// Attention of beams over a paged cache, one query token a beam.
//
//   out_i = softmax(q_i K_i' scale) V_i over the first kv_len[i] keys of beam i; scores, maximum and sum in float32, weights
//   rounded to bfloat16 for the product with V, whose accumulators are float32.
//
// Beams of a request hold the same pages up to where they parted.  The rows of a tile are the (beam, query head) pairs of one key
// head, so that a shared page is read once for all beams; behind it every beam's own pages follow, one beam after another, for
// the rows of that beam alone.  A softmax over a union of keys joins from (maximum, sum, weighted values), whoever made the parts.
//
// Bound by the bytes of the keys.  The work is a flat list: a request's block of rows, its key heads, their units of 32 keys.  Every
// team of warps has an even, consecutive share of it: the copy engine brings its units (128-byte swizzle) into a ring of the team's
// own, ahead across the ends of requests.  A warp has 16 rows; a team is as many warps as the rows need, up to eight, all on the same
// units, the first of which asks for them.  Warp-level products (mma.sync): a request's rows are an eighth to a half of a
// tensor-core tile.  Where a share ends inside a block of rows, the sums go out as a partial result; a second launch joins those.
#include <math_constants.h>
#include <stdio.h>

#include "tc_common.cuh"

namespace {

typedef __nv_bfloat16 bf16;

constexpr int PAGE = 64, KEYS = 32;                // keys of a page, of a unit
constexpr int MOST_BEAMS = 32;
constexpr float RESCALE_LOG2 = 8.0f;               // weights may grow to 2^8 before what was summed up is scaled down
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  const bf16* q;
  bf16* out;
  float* part_o;       // [teams][2][rows of a team][hd], not divided by their sums; of a share's first rows (0) and last rows (1)
  float2* part_ml;     // ... maximum (in units of log2), sum
  int2* parts;         // [beams][heads]: first team with a part of the row, number of teams
  const int* table;
  const int* kv_len;
  const int* shared;
  int R, K, nh, nkv, hd, W, n_pages;
  int team, row_blocks, fewest;                    // warps of a team; blocks of rows of a request; units of a share at least
  float scale_log2;
};

constexpr int ROWS = 16;                           // of a warp

template <int HDC>
struct Shape {
  static constexpr int SLABS = HDC / 64, SLAB = KEYS * 128;                // 64 numbers of the keys of a unit
  static constexpr int TILE = SLABS * SLAB, STAGE = 2 * TILE;              // keys, values
  static constexpr int STAGES = HDC > 128 ? 6 : 12, RING = STAGES * STAGE;
  // queries lie in registers, as the products take them, where results leave room for them
  static constexpr bool Q_REGS = HDC <= 128;
  static constexpr int Q_SLAB = ROWS * 128, Q = Q_REGS ? 0 : SLABS * Q_SLAB;
  static constexpr int WARPS = HDC > 128 ? 4 : 8, THREADS = 32 * WARPS;   // at most
  static constexpr int Q_WARPS = 4;                                        // (at most, where queries lie in shared memory)
  static constexpr int SMEM = RING + Q_WARPS * Q + STAGES * 24;            // ... and two barriers and a unit's description a stage
  static_assert(SMEM <= 227 * 1024, "shared memory of a block");
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bounded wait: false (and *status = code) if the phase did not complete in 4e9 cycles, about two seconds.
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
  int units;
  int len, first, own, upto;        // of the lane's beam: keys, first page of its own, units of its own, of the beams up to it
};

__device__ __forceinline__ Rows look_up(const Args& a, int block) {
  const int lane = threadIdx.x & 31, G = a.nh / a.nkv, all = ROWS * a.team;
  Rows x;
  x.request = block / a.row_blocks;
  x.rho0 = block % a.row_blocks * all;
  x.n_rows = min(all, a.K * G - x.rho0);
  x.len = lane < a.K ? min(max(a.kv_len[x.request * a.K + lane], 0), a.W * PAGE) : 0;
  const int most = __reduce_max_sync(0xffffffffu, x.len);
  x.head = __ffs(__ballot_sync(0xffffffffu, lane < a.K && x.len == most)) - 1;
  x.common = min(max(a.shared[x.request], 0), most / PAGE);
  x.first = x.len < x.common * PAGE ? 0 : x.common;        // shorter beams read all they have by themselves
  x.own = lane >= x.rho0 / G && lane <= (x.rho0 + x.n_rows - 1) / G ? (x.len - x.first * PAGE + KEYS - 1) / KEYS : 0;
  x.upto = x.own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, x.upto, o);
    if (lane >= o) x.upto += t;
  }
  x.units = max(1, x.common * (PAGE / KEYS) + __shfl_sync(0xffffffffu, x.upto, 31));     // (rows without keys have a unit as well)
  return x;
}
// The units of a block, by one thread.
__device__ __forceinline__ int count_units(const Args& a, int block) {
  const int G = a.nh / a.nkv, all = ROWS * a.team, r = block / a.row_blocks, rho0 = block % a.row_blocks * all;
  const int beam0 = rho0 / G, beam1 = (min(rho0 + all, a.K * G) - 1) / G;
  int most = 0;
#pragma unroll 4
  for (int k = 0; k < a.K; ++k) most = max(most, min(max(a.kv_len[r * a.K + k], 0), a.W * PAGE));
  const int common = min(max(a.shared[r], 0), most / PAGE);
  int n = common * (PAGE / KEYS);
#pragma unroll 4
  for (int k = beam0; k <= beam1; ++k) {
    const int len = min(max(a.kv_len[r * a.K + k], 0), a.W * PAGE);
    n += (len - (len < common * PAGE ? 0 : common * PAGE) + KEYS - 1) / KEYS;
  }
  return max(1, n);
}

// A place of the list as one thread walks it: the unit's beam (-1: all that share it), its first key, and where its page stands.
struct Cursor {
  int block, kvh, unit, units, shared_units;
  int request, head, common, beam0, beam1;
  int beam, at, keys;
  const int* entry;                 // of the table; null: a unit without keys

  __device__ __forceinline__ int length(const Args& a, int b) const { return min(max(a.kv_len[request * a.K + b], 0), a.W * PAGE); }
  __device__ __forceinline__ int own_from(int len) const { return len < common * PAGE ? 0 : common * PAGE; }
  __device__ __forceinline__ void enter(const Args& a, int to) {
    const int G = a.nh / a.nkv, all = ROWS * a.team, rho0 = to % a.row_blocks * all;
    block = to, request = to / a.row_blocks, beam0 = rho0 / G, beam1 = (min(rho0 + all, a.K * G) - 1) / G;
    int most = -1;
    head = 0;
    for (int k = 0; k < a.K; ++k) {
      const int len = length(a, k);
      if (len > most) most = len, head = k;
    }
    common = min(max(a.shared[request], 0), most / PAGE);
    units = shared_units = common * (PAGE / KEYS);
    for (int k = beam0; k <= beam1; ++k) {
      const int len = length(a, k);
      units += (len - own_from(len) + KEYS - 1) / KEYS;
    }
    units = max(1, units);
  }
  __device__ __forceinline__ void find(const Args& a) {      // the unit's keys
    if (unit < shared_units) {
      beam = -1, at = unit * KEYS, keys = KEYS;
      entry = a.table + ((size_t)request * a.K + head) * a.W + at / PAGE;
      return;
    }
    int left = unit - shared_units;
    for (beam = beam0; beam <= beam1; ++beam) {
      const int len = length(a, beam), from = own_from(len), own = (len - from + KEYS - 1) / KEYS;
      if (left < own) {
        at = from + left * KEYS, keys = min(KEYS, len - at);
        entry = a.table + ((size_t)request * a.K + beam) * a.W + at / PAGE;
        return;
      }
      left -= own;
    }
    beam = -1, at = keys = 0, entry = nullptr;
  }
  __device__ __forceinline__ void step(const Args& a) {
    if (++unit == units) {
      unit = 0;
      if (++kvh == a.nkv) kvh = 0, enter(a, block + 1);
    } else if (beam >= 0 && at + KEYS < length(a, beam)) {  // the next keys of the same beam
      entry += (at % PAGE + KEYS) / PAGE;
      at += KEYS;
      keys = min(KEYS, length(a, beam) - at);
      return;
    }
    find(a);
  }
};

template <int HDC>
__global__ void __launch_bounds__(Shape<HDC>::THREADS, HDC <= 64 ? 2 : 1) beam_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                             const Args a, int* __restrict__ status) {
  typedef Shape<HDC> C;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, hd = a.hd, G = a.nh / a.nkv;
  const int T = a.team, here = blockDim.x / 32 / T, team = warp / T, member = warp % T, stages = C::STAGES / here;
  const uint32_t base = jb::smem_u32(smem), ring = base + team * stages * C::STAGE;
  const uint32_t bars = base + C::RING + C::Q_WARPS * C::Q + team * stages * 16;   // of a stage: full, empty
  int2* about = reinterpret_cast<int2*>(smem + C::RING + C::Q_WARPS * C::Q + C::STAGES * 16) + team * stages;   // keys, beam
  if (member == 0 && lane == 0) {
    for (int i = 0; i < stages; ++i) jb::mbar_init(bars + 16 * i, 1), jb::mbar_init(bars + 16 * i + 8, T);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  // ---- the list's length, and this team's share ----
  const int blocks = a.R * a.row_blocks, chunk = (blocks + 31) / 32, block0 = min(lane * chunk, blocks), block1 = min(block0 + chunk, blocks);
  int mine = 0;
  for (int i = block0; i < block1; ++i) mine += count_units(a, i);
  mine *= a.nkv;
  int up = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += t;
  }
  const int total = __shfl_sync(0xffffffffu, up, 31), teams = gridDim.x * here, worker = blockIdx.x * here + team;
  const int per = max(a.fewest, (total + teams - 1) / teams);
  const int begin = min(worker * per, total), end = min(begin + per, total);
  if (begin >= end) return;                                // (a whole team)
  Rows x;
  int block, kvh, unit;                                    // the place of the list
  {
    const int owner = __ffs(__ballot_sync(0xffffffffu, begin < up)) - 1;
    int before = __shfl_sync(0xffffffffu, up - mine, owner);
    for (block = owner * chunk;; ++block) {
      x = look_up(a, block);
      if (begin < before + x.units * a.nkv) break;
      before += x.units * a.nkv;
    }
    kvh = (begin - before) / x.units;
    unit = begin - before - kvh * x.units;
  }
  // ---- the team's first warp asks for units, ahead across the ends of rows ----
  Cursor u{};
  int page = -1, asked = begin, asked_stage = 0;
  if (member == 0) {
    u.enter(a, block);
    u.kvh = kvh, u.unit = unit;
    u.find(a);
    page = u.entry != nullptr ? *u.entry : -1;
  }
  auto issue = [&]() {
    if (lane == 0) {
      const bool there = page >= 0 && page < a.n_pages;     // (no page: no keys)
      const int row = ((there ? page : 0) * a.nkv + u.kvh) * PAGE + u.at % PAGE;
      about[asked_stage] = make_int2(there ? u.keys : 0, u.beam);
      const uint32_t full = bars + 16 * asked_stage, to = ring + asked_stage * C::STAGE;
      jb::mbar_expect_tx(full, C::STAGE);                   // (behind the head's numbers the copy engine writes zeroes)
#pragma unroll
      for (int h = 0; h < C::SLABS; ++h) jb::tma_load_2d(to + h * C::SLAB, &map_k, full, h * 64, row);
#pragma unroll
      for (int h = 0; h < C::SLABS; ++h) jb::tma_load_2d(to + C::TILE + h * C::SLAB, &map_v, full, h * 64, row);
    }
    __syncwarp();
    if (++asked_stage == stages) asked_stage = 0;
    if (++asked < end) {                                    // (a unit's page is looked up a turn before it is asked for)
      u.step(a);
      page = u.entry != nullptr ? *u.entry : -1;
    }
  };
  if (member == 0)
    for (int i = 0; i < stages && asked < end; ++i) issue();
  // Places of the operands in swizzled rows: 16 bytes `piece` of row r lie at piece ^ (r % 8), so that a step of 32 bytes is an
  // exclusive or.
  const int c = lane & 3, r8 = lane & 7;
  const uint32_t k_lane = (r8 + ((lane >> 4) << 3)) * 128 + ((((lane >> 3) & 1) ^ r8) << 4);
  const uint32_t v_lane = (lane & 15) * 128 + (((lane >> 4) ^ r8) << 4);
  const uint32_t q_at = base + C::RING + warp * C::Q;
  int beam_of[2] = {-1, -1};         // of this thread's rows; -1: no row
  bool joins[2] = {false, false};    // whether the row reads the shared pages
  bool all_join = false;
  int beam_first = 0, beam_last = -1;     // of the warp's rows
  float m[2], l[2], o[HDC / 8][4];
  uint32_t q[C::Q_REGS ? HDC / 16 : 1][4];
  bool ok = true;
  int st = 0, st_before = 0;
  uint32_t phase = 0, phase_before = 0;
  for (int i = begin; i < end; ++i) {
    if (i > begin && member == 0 && asked < end) {         // the stage of the turn before, when all warps are done with it
      ok = __all_sync(0xffffffffu, mbar_wait(bars + 16 * st_before + 8, phase_before, status, 54));
      if (!ok) break;
      issue();
    }
    if (i == begin || unit == 0) {
      const int row0 = member * ROWS, rho0 = x.rho0 + row0, n_rows = min(ROWS, x.n_rows - row0);
      beam_first = rho0 / G, beam_last = n_rows > 0 ? (rho0 + n_rows - 1) / G : -1;
      bool every = true;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = (lane >> 2) + 8 * h;
        const bool valid = row < n_rows;
        beam_of[h] = valid ? (rho0 + row) / G : -1;
        const int len = __shfl_sync(0xffffffffu, x.len, max(beam_of[h], 0));
        joins[h] = valid && len >= x.common * PAGE;
        every = every && (joins[h] || !valid);
        m[h] = -CUDART_INF_F;
        l[h] = 0.0f;
        if constexpr (C::Q_REGS) {
          const bf16* src = a.q + (((size_t)x.request * a.K + max(beam_of[h], 0)) * a.nh + kvh * G + (valid ? (rho0 + row) % G : 0)) * hd + 2 * c;
#pragma unroll
          for (int ks = 0; ks < HDC / 16; ++ks)
#pragma unroll
            for (int half = 0; half < 2; ++half)
              q[ks][h + 2 * half] = valid && ks * 16 + half * 8 < hd ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + half * 8) : 0u;
        }
      }
      if constexpr (!C::Q_REGS) {
        for (int ch = lane; ch < ROWS * C::SLABS * 8; ch += 32) {
          const int row = ch / (C::SLABS * 8), piece = ch % (C::SLABS * 8), rho = rho0 + row;
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (row < n_rows && piece * 8 < hd)
            v = *reinterpret_cast<const uint4*>(a.q + (((size_t)x.request * a.K + rho / G) * a.nh + kvh * G + rho % G) * hd + piece * 8);
          *reinterpret_cast<uint4*>(smem + C::RING + warp * C::Q + (piece / 8) * C::Q_SLAB + row * 128 + (((piece % 8) ^ (row & 7)) << 4)) = v;
        }
      }
#pragma unroll
      for (int j = 0; j < HDC / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
      all_join = __all_sync(0xffffffffu, every);           // (rows behind the last may do as they like)
      __syncwarp();
    }
    ok = __all_sync(0xffffffffu, mbar_wait(bars + 16 * st, phase, status, 53));
    if (!ok) break;
    const int2 info = about[st];
    const int keys = info.x, beam = info.y;
    const uint32_t k_t = ring + st * C::STAGE, v_t = k_t + C::TILE;
    // (units of another warp's beams are nothing to this one)
    if (keys > 0 && (beam < 0 ? beam_last >= 0 : beam >= beam_first && beam <= beam_last)) {
      if (keys < KEYS) {                                   // values behind the last key: a weight of 0 does not silence what is no number
        for (int p = lane; p < (KEYS - keys) * C::SLABS * 8; p += 32) {
          const int row = keys + p / (C::SLABS * 8), piece = p % (C::SLABS * 8);
          *reinterpret_cast<uint4*>(smem + (v_t - base) + (piece / 8) * C::SLAB + row * 128 + ((piece % 8) << 4)) = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
      }
      float s[4][4], s_odd[4][4];                          // (two chains of products, a half as long each)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = s_odd[j][e] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < HDC / 16; ++ks) {
        uint32_t qa[4], b[2][4];
        const uint32_t at = k_t + (k_lane ^ ((ks % 4) << 5)) + (ks / 4) * C::SLAB;
        ldmatrix_x4(b[0], at);
        ldmatrix_x4(b[1], at + 16 * 128);
        if constexpr (C::Q_REGS) {
#pragma unroll
          for (int e = 0; e < 4; ++e) qa[e] = q[ks][e];
        } else {
          ldmatrix_x4(qa, q_at + (v_lane ^ ((ks % 4) << 5)) + (ks / 4) * C::Q_SLAB);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mma_bf16(ks & 1 ? s_odd[2 * j] : s[2 * j], qa, b[j][0], b[j][1]);
          mma_bf16(ks & 1 ? s_odd[2 * j + 1] : s[2 * j + 1], qa, b[j][2], b[j][3]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] += s_odd[j][e];
      if (beam >= 0 || keys < KEYS || !all_join) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int h = e >> 1, key = j * 8 + 2 * c + (e & 1);
            if (!(key < keys && (beam < 0 ? joins[h] : beam_of[h] == beam))) s[j][e] = -CUDART_INF_F;
          }
      }
      float mx[2], use[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        mx[h] = fmaxf(fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1])),
                      fmaxf(fmaxf(s[2][2 * h], s[2][2 * h + 1]), fmaxf(s[3][2 * h], s[3][2 * h + 1]))) * a.scale_log2;
      // what weights are relative to is raised only when a score passes it by RESCALE_LOG2 (also the first number of all)
      if (__any_sync(0xffffffffu, mx[0] > m[0] + RESCALE_LOG2 || mx[1] > m[1] + RESCALE_LOG2)) {
        float corr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
          const float top = fmaxf(m[h], mx[h]);
          corr[h] = top == -CUDART_INF_F ? 1.0f : fast_exp2(m[h] - top);
          m[h] = top;
          l[h] *= corr[h];
        }
#pragma unroll
        for (int j = 0; j < HDC / 8; ++j) o[j][0] *= corr[0], o[j][1] *= corr[0], o[j][2] *= corr[1], o[j][3] *= corr[1];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) use[h] = m[h] == -CUDART_INF_F ? 0.0f : m[h];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = fast_exp2(fmaf(s[j][e], a.scale_log2, -use[e >> 1]));
#pragma unroll
      for (int h = 0; h < 2; ++h)
        l[h] += ((s[0][2 * h] + s[0][2 * h + 1]) + (s[1][2 * h] + s[1][2 * h + 1])) + ((s[2][2 * h] + s[2][2 * h + 1]) + (s[3][2 * h] + s[3][2 * h + 1]));
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const uint32_t pa[4] = {pack_bf16(s[2 * kk][0], s[2 * kk][1]), pack_bf16(s[2 * kk][2], s[2 * kk][3]),
                                pack_bf16(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack_bf16(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
        for (int j = 0; j < HDC / 8; j += 2) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, v_t + (v_lane ^ ((j % 8) << 4)) + (j / 8) * C::SLAB + kk * 16 * 128);
          mma_bf16(o[j], pa, b[0], b[1]);
          mma_bf16(o[j + 1], pa, b[2], b[3]);
        }
      }
      if (keys < KEYS) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // zeroes, before the copy engine writes there again
    }
    __syncwarp();
    if (lane == 0) jb::mbar_arrive(bars + 16 * st + 8);
    st_before = st, phase_before = phase;
    if (++st == stages) st = 0, phase ^= 1;
    if (unit + 1 == x.units || i + 1 == end) {             // the rows' keys end here, or the share does
      const int start = i - unit, first = start / per, last = (start + x.units - 1) / per;
      const bool complete = first == last;
      const size_t record = ((size_t)worker * 2 + (worker == first ? 1 : 0)) * (ROWS * T) + member * ROWS;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = l[h];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int row = (lane >> 2) + 8 * h, rho = x.rho0 + member * ROWS + row;
        if (beam_of[h] < 0) continue;
        const size_t item = ((size_t)x.request * a.K + beam_of[h]) * a.nh + kvh * G + rho % G;
        if (c == 0) {
          if (worker == first) a.parts[item] = make_int2(first, last - first + 1);
          if (!complete) a.part_ml[record + row] = make_float2(m[h], sum);
        }
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
        for (int j = 0; j < HDC / 8; ++j) {
          if (j * 8 < hd) {
            if (complete) *reinterpret_cast<uint32_t*>(a.out + item * hd + j * 8 + 2 * c) = pack_bf16(o[j][2 * h] * inv, o[j][2 * h + 1] * inv);
            else *reinterpret_cast<float2*>(a.part_o + (record + row) * hd + j * 8 + 2 * c) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
          }
        }
      }
    }
    if (++unit == x.units) {
      unit = 0;
      if (++kvh == a.nkv) {
        kvh = 0;
        if (i + 1 < end) x = look_up(a, ++block);
      }
    }
  }
  // gave up: what is still on its way arrives before the block ends (or its wait gives up as well)
  if (!ok && member == 0)
    for (int turn = max(0, asked - begin - stages); turn < asked - begin; ++turn) mbar_wait(bars + 16 * (turn % stages), (turn / stages) & 1, status, 53);
}

// A warp a (beam, head): the parts of its keys joined, where there are several.
__global__ void __launch_bounds__(128) beam_attention_join_kernel(const Args a, int rows) {
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, G = a.nh / a.nkv;
  if (item >= (long long)a.R * a.K * a.nh) return;
  const int2 parts = a.parts[item];
  if (parts.y <= 1) return;
  const int head = (int)(item % a.nh), beam = (int)(item / a.nh % a.K), row = (beam * G + head % G) % rows;
  auto record = [&](int p) { return ((size_t)(parts.x + p) * 2 + (p == 0 ? 1 : 0)) * rows + row; };
  float most = -CUDART_INF_F;
  for (int p = lane; p < parts.y; p += 32) most = fmaxf(most, a.part_ml[record(p)].x);
  most = jb::warp_max(most);
  const float use = most == -CUDART_INF_F ? 0.0f : most;
  for (int d = lane * 4; d < a.hd; d += 128) {
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
#pragma unroll 4
    for (int p = 0; p < parts.y; ++p) {
      const float2 ml = a.part_ml[record(p)];
      const float4 v = *reinterpret_cast<const float4*>(a.part_o + record(p) * a.hd + d);
      const float f = fast_exp2(ml.x - use);
      sum = fmaf(f, ml.y, sum);
      o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    *reinterpret_cast<uint2*>(a.out + item * a.hd + d) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
  }
}

template <int HDC>
cudaError_t go(const CUtensorMap* maps, Args a, int blocks, int warps, int* status, cudaStream_t stream) {
  typedef Shape<HDC> C;
  static bool ready[64] = {};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= 64 || !ready[device]) {
    e = cudaFuncSetAttribute(beam_attention_kernel<HDC>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    if (device < 64) ready[device] = true;
  }
  jb::Launch cfg(dim3(blocks), dim3(32 * warps), C::SMEM, stream);
  e = cudaLaunchKernelEx(&cfg.c, beam_attention_kernel<HDC>, maps[0], maps[1], a, status);
  if (e != cudaSuccess) return e;
  jb::Launch join(dim3((unsigned)(((long long)a.R * a.K * a.nh + 3) / 4)), dim3(128), 0, stream);
  return cudaLaunchKernelEx(&join.c, beam_attention_join_kernel, a, ROWS * a.team);
}

}  // namespace

// part: float32 scratch of blocks * warps * 16 * 2 (hd + 2) + 2 R K nh numbers.  blocks, warps of a block, team (warps that work on the same
// units, a divisor of them): see `ops.beam_attention_plan`.
JB_EXPORT int jb_attention_beams(const void* q, const void* k_cache, const void* v_cache, void* out, void* part, const int* table,
                                 const int* kv_len, const int* shared, int R, int K, int nh, int nkv, int hd, int W, int n_pages, int blocks,
                                 int warps, int team, int fewest, float scale, int* status, cudaStream_t stream) {
  JB_REFUSE(R < 1 || K < 1 || K > MOST_BEAMS || nkv < 1 || nh < nkv || nh % nkv || hd < 8 || hd > 256 || hd % 8 || W < 1 || W > 0x7fffffff / PAGE ||
                n_pages < 1 || (long long)n_pages * nkv * PAGE > 0x7fffffffLL || blocks < 1 || fewest < 1 || team < 1 || warps < team ||
                warps % team || warps > (hd > 128 ? Shape<256>::WARPS : Shape<128>::WARPS) || warps / team > (hd > 128 ? 3 : 6) || !(scale > 0.0f),
            "attention_beams: %d groups of %d beams, %d heads over %d of %d numbers, %d pages a row of %d, plan %d %d %d %d, scale %g", R, K, nh,
            nkv, hd, W, n_pages, blocks, warps, team, fewest, scale);
  CUtensorMap maps[2];
  if (!jb::make_map_64(&maps[0], k_cache, (uint64_t)n_pages * nkv * PAGE, hd, KEYS, true) ||
      !jb::make_map_64(&maps[1], v_cache, (uint64_t)n_pages * nkv * PAGE, hd, KEYS, true))
    return JB_ERR_TENSORMAP;
  Args a{};
  a.q = (const bf16*)q, a.out = (bf16*)out, a.table = table, a.kv_len = kv_len, a.shared = shared;
  const size_t records = (size_t)blocks * warps * ROWS * 2;
  a.part_o = (float*)part, a.part_ml = (float2*)(a.part_o + records * hd), a.parts = (int2*)(a.part_ml + records);
  a.R = R, a.K = K, a.nh = nh, a.nkv = nkv, a.hd = hd, a.W = W, a.n_pages = n_pages;
  a.team = team, a.fewest = fewest, a.scale_log2 = scale * LOG2E;
  a.row_blocks = (K * (nh / nkv) + ROWS * team - 1) / (ROWS * team);
  return (int)(hd > 128 ? go<256>(maps, a, blocks, warps, status, stream) : hd > 64 ? go<128>(maps, a, blocks, warps, status, stream)
                                                                               : go<64>(maps, a, blocks, warps, status, stream));
}
