// The index arrays of a step, made on the device from request lengths: pages are taken from the free list and given back,
// and every new token gets its position, its request and its cache row.
//
// With page size p, width W of a block table and P shared pages in front of every row, request b has
//   kv_len = length + new,   held0 = P if it begins, else the pages of the row it goes on with,
//   need   = max(0, min(ceil(kv_len / p), W) - held0).
// The pool is the free list followed by the pages (behind the shared ones) of the rows nobody goes on with, row after row;
// request b takes pool[E_b, E_b + need_b) with E the exclusive sum of need, and what is left over is the next free list.
// The same lists give the same tables whatever the launch looks like: there are no atomics but on a bitmap.
//
// One launch, bound by how often it waits for memory: 3.9 us for 4 requests, 4.8 for 256, 9.7 for 1,024 of up to 512 pages each.  Every
// block makes the three sums (new tokens, pages needed, pages given back) by itself in shared memory, in one pass, which costs less
// than a second launch or a wait between blocks.  Then table rows, tokens and free pages each have blocks of their own: made one list
// after another by the same threads their waits added up (256 requests: 8.3 us, with three passes for the sums).
#include <stddef.h>
#include <stdio.h>
#include <string.h>

#include "common.cuh"

namespace {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int SMS = 148;

struct Args {
  const int* lengths;
  const int* fresh;       // new tokens of each request
  const int* rows;        // row of the old table that a request goes on with; anything outside it: the request begins
  const int* old_table;
  const int* old_held;
  const int* prefix;
  const int* free_pages;
  const int* n_free;
  int* q_start;
  int* kv_len;
  int* positions;
  int* token_seq;
  int* dest;
  int* table;
  int* held;
  int* free_out;
  int* n_free_out;
  int* missing;
  int B, B0, T, W0, W, P, N, page_size;
  int blocks[3];          // that make table rows, tokens, free pages
};

__device__ __forceinline__ int pages_of(int tokens, int page_size) { return tokens / page_size + (tokens % page_size != 0); }

// The largest i with sums[i] <= x, of sums[0 .. n] rising, sums[0] <= x < sums[n].
__device__ __forceinline__ int owner(const int* sums, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(THREADS) step_tables_kernel(const Args a) {
  extern __shared__ int smem[];
  __shared__ int warp_sum[3][WARPS];
  int* starts = smem;                     // [B + 1] first token of each request
  int* takes = starts + a.B + 1;          // [B + 1] first place of the pool that each request takes
  int* gives = takes + a.B + 1;           // [B0 + 1] first given-back place of each old row
  unsigned* goes_on = (unsigned*)(gives + a.B0 + 1);   // a bit for each old row
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  const int width = min(a.W0, a.W);
  for (int i = threadIdx.x; i < (a.B0 + 31) / 32; i += THREADS) goes_on[i] = 0u;
  __syncthreads();
  auto row_of = [&](int b) {
    const int r = a.rows[b];
    return r >= 0 && r < a.B0 ? r : -1;
  };
  auto held_of = [&](int r) { return min(max(a.old_held[r], 0), width); };
  auto held_before = [&](int r) { return r < 0 ? min(a.P, a.W) : held_of(r); };
  auto length_of = [&](int b) { return max(a.lengths[b], 0); };
  auto fresh_of = [&](int b) { return max(a.fresh[b], 0); };
  // ---- the sums: what a thread needs of the first THREADS requests and rows is asked for at once ----
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  struct Item {
    int length, fresh, row, held;   // of request i; the pages that old row i holds
  };
  auto load = [&](int i) {
    Item x{0, 0, -1, 0};
    if (i < a.B) x.length = length_of(i), x.fresh = fresh_of(i), x.row = row_of(i);
    if (i < a.B0) x.held = held_of(i);
    return x;
  };
  Item x = load(threadIdx.x);
  const int listed = min(max(*a.n_free, 0), a.N);
  for (int i = threadIdx.x; i < a.B; i += THREADS) {
    const int r = i == threadIdx.x ? x.row : row_of(i);
    if (r >= 0) atomicOr(&goes_on[r >> 5], 1u << (r & 31));
  }
  int before = threadIdx.x < a.B ? held_before(x.row) : 0;
  __syncthreads();
  int carry[3] = {0, 0, 0};
  for (int i0 = 0; i0 < max(a.B, a.B0); i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    if (i0 > 0) {
      x = load(i);
      before = i < a.B ? held_before(x.row) : 0;
    }
    int v[3] = {0, 0, 0}, up[3];
    if (i < a.B) v[0] = x.fresh, v[1] = max(0, min(pages_of(x.length + x.fresh, a.page_size), a.W) - before);
    if (i < a.B0 && !((goes_on[i >> 5] >> (i & 31)) & 1u)) v[2] = max(0, x.held - a.P);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      up[k] = v[k];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, up[k], o);
        if (lane >= o) up[k] += t;
      }
      if (lane == 31) warp_sum[k][warp] = up[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int in_front = carry[k];
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w == warp) in_front = carry[k];
        carry[k] += warp_sum[k][w];
      }
      int* out = k == 0 ? starts : k == 1 ? takes : gives;
      if (i < (k < 2 ? a.B : a.B0)) out[i] = in_front + up[k] - v[k];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) starts[a.B] = carry[0], takes[a.B] = carry[1], gives[a.B0] = carry[2];
  __syncthreads();
  const int n_free = listed;
  const int have = n_free + gives[a.B0], took = min(takes[a.B], have), left = have - took;
  auto pool = [&](int i) {
    if (i < n_free) return a.free_pages[i];
    const int r = owner(gives, a.B0, i - n_free);
    return a.old_table[(size_t)r * a.W0 + a.P + (i - n_free - gives[r])];
  };
  auto page_at = [&](int b, int r, int held0, int c) {
    if (c < held0) return r < 0 ? a.prefix[c] : a.old_table[(size_t)r * a.W0 + c];
    const int i = takes[b] + c - held0;
    return i < takes[b + 1] && i < have ? pool(i) : -1;
  };
  // ---- the outputs: table rows, tokens, free pages, each by blocks of their own, as a thread's would follow one another ----
  const int kind = blockIdx.x < a.blocks[0] ? 0 : blockIdx.x < a.blocks[0] + a.blocks[1] ? 1 : 2;
  const int first = kind == 0 ? 0 : kind == 1 ? a.blocks[0] : a.blocks[0] + a.blocks[1];
  const int thread = (blockIdx.x - first) * THREADS + threadIdx.x, threads = a.blocks[kind] * THREADS;
  if (kind == 0) {
    for (int b = thread >> 5; b < a.B; b += threads >> 5) {
      const int r = row_of(b), held0 = held_before(r);
      int* row = a.table + (size_t)b * a.W;
      for (int c = lane; c < a.W; c += 32) row[c] = page_at(b, r, held0, c);
      if (lane == 0) {
        a.kv_len[b] = length_of(b) + fresh_of(b);
        a.held[b] = held0 + max(0, min(takes[b + 1], have) - min(takes[b], have));
      }
    }
    return;
  }
  if (kind == 1) {
    for (int t = thread; t < a.T; t += threads) {
      int position = -1, b = -1, dest = -1;
      if (t < starts[a.B]) {
        b = owner(starts, a.B, t);
        position = length_of(b) + t - starts[b];
        const int c = position / a.page_size, r = row_of(b);
        const int page = c < a.W ? page_at(b, r, held_before(r), c) : -1;
        if (page >= 0) dest = page * a.page_size + position % a.page_size;
      }
      a.positions[t] = position;
      a.token_seq[t] = b;
      a.dest[t] = dest;
    }
    return;
  }
  for (int i = thread; i < a.N; i += threads) a.free_out[i] = i < left ? pool(took + i) : -1;
  for (int b = thread; b <= a.B; b += threads) a.q_start[b] = starts[b];
  if (blockIdx.x == first) {
    int over = 0;
    for (int b = threadIdx.x; b < a.B; b += THREADS) over += max(0, pages_of(length_of(b) + fresh_of(b), a.page_size) - a.W);
    over = __reduce_add_sync(0xffffffffu, over);
    if (lane == 0) warp_sum[0][warp] = over;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < WARPS; ++w) over += warp_sum[0][w];
      *a.missing = takes[a.B] - took + over + max(0, left - a.N);   // (what the new list has no place for is lost)
      *a.n_free_out = min(left, a.N);
    }
  }
}

// Whether one of the ten outputs lies over one of the eight inputs or over another output, wherever each begins (inputs may share places).
bool made_over_others(const Args& a) {
  const char* at[18];
  static_assert(offsetof(Args, B) == sizeof(at), "18 tensors, the inputs first");
  memcpy(at, &a, sizeof(at));
  const size_t n[18] = {(size_t)a.B, (size_t)a.B, (size_t)a.B, (size_t)a.B0 * a.W0, (size_t)a.B0, (size_t)a.P, (size_t)a.N, 1, (size_t)a.B + 1, (size_t)a.B,
                        (size_t)a.T, (size_t)a.T, (size_t)a.T, (size_t)a.B * a.W, (size_t)a.B, (size_t)a.N, 1, 1};
  for (int i = 8; i < 18; ++i)
    for (int j = 0; j < i; ++j)
      if (n[i] > 0 && n[j] > 0 && at[i] < at[j] + 4 * n[j] && at[j] < at[i] + 4 * n[i]) return true;
  return false;
}

size_t smem_for(int B, int B0) { return (size_t)(2 * (B + 1) + B0 + 1 + (B0 + 31) / 32) * sizeof(int); }

}  // namespace

// given: an Args without its last member, in host memory (18 pointers one by one cost the host as much as a launch).  Every pointer
// is device memory of int32; outputs overlap no input.  n_free_out, missing: one int each.
JB_EXPORT int jb_step_tables(const void* given, cudaStream_t stream) {
  static_assert(offsetof(Args, blocks) == 18 * 8 + 8 * 4, "as the caller packs it");
  Args a{};
  memcpy(&a, given, offsetof(Args, blocks));
  const int B = a.B, B0 = a.B0, T = a.T, W0 = a.W0, W = a.W, P = a.P, N = a.N, page_size = a.page_size;
  JB_REFUSE(B < 0 || B0 < 0 || T < 0 || W <= 0 || W0 < 0 || P < 0 || N < 0 || page_size <= 0, "step_tables: sizes %d %d %d %d %d %d %d %d", B, B0,
            T, W, W0, P, N, page_size);
  JB_REFUSE(W < W0 || P > W, "step_tables: a table of %d pages a row cannot take over rows of %d behind %d shared pages", W, W0, P);
  if (made_over_others(a)) return JB_ERR_OVERLAP;
  const size_t smem = smem_for(B, B0);
  JB_REFUSE(smem > 200 * 1024, "step_tables: %d requests after %d are more than a block's memory holds sums of", B, B0);
  if (smem > 48 * 1024) {
    static size_t allowed = 48 * 1024;
    if (smem > allowed) {
      cudaError_t e = cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return (int)e;
      allowed = smem;
    }
  }
  // A block for THREADS places of a list, but about one a multiprocessor in all, shared by the lists' work: more blocks make the sums more
  // often (1,024 requests of up to 512 pages: 9.7 us, 12.4 by 148 blocks a list).  A token, whose request is searched for, is as much
  // work as four places of the table.
  const long long items[3] = {(long long)B * W, T, N}, all = items[0] + 4 * items[1] + items[2];
  int blocks = 0;
  for (int k = 0; k < 3; ++k) {
    const long long wanted = (items[k] + THREADS - 1) / THREADS, share = all > 0 ? items[k] * (k == 1 ? 4 : 1) * SMS / all : 0;
    const long long n = wanted < share || wanted <= SMS / 3 ? wanted : share;
    a.blocks[k] = n < 1 ? 1 : (int)n;
    blocks += a.blocks[k];
  }
  jb::Launch cfg(dim3(blocks), dim3(THREADS), smem, stream);
  return (int)cudaLaunchKernelEx(&cfg.c, step_tables_kernel, a);
}
