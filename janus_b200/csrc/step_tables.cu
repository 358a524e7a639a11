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
// One launch.  Every block makes the three sums (new tokens, pages needed, pages given back) by itself in shared memory, which
// costs less than a second launch or a wait between blocks: 1,024 requests are one to four elements a thread.  Then the blocks
// share the outputs out among themselves.
#include <stdio.h>

#include "common.cuh"

namespace {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;

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
};

__device__ __forceinline__ int pages_of(int tokens, int page_size) { return tokens / page_size + (tokens % page_size != 0); }

// Exclusive sums of n values, value(i) for i < n, into out[0 .. n] (out[n]: the sum of all).  `warp_sum`: WARPS ints.
template <typename F>
__device__ __forceinline__ void exclusive_sums(F&& value, int n, int* out, int* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int carry = 0;
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    const int v = i < n ? value(i) : 0;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int before = carry, all = carry;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w == warp) before = all;
      all += warp_sum[w];
    }
    if (i < n) out[i] = before + s - v;
    carry = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) out[n] = carry;
}

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
  __shared__ int warp_sum[WARPS];
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
  for (int b = threadIdx.x; b < a.B; b += THREADS) {
    const int r = row_of(b);
    if (r >= 0) atomicOr(&goes_on[r >> 5], 1u << (r & 31));
  }
  __syncthreads();
  exclusive_sums([&](int b) { return fresh_of(b); }, a.B, starts, warp_sum);
  exclusive_sums(
      [&](int b) {
        const int want = min(pages_of(length_of(b) + fresh_of(b), a.page_size), a.W);
        return max(0, want - held_before(row_of(b)));
      },
      a.B, takes, warp_sum);
  exclusive_sums([&](int r) { return (goes_on[r >> 5] >> (r & 31)) & 1u ? 0 : max(0, held_of(r) - a.P); }, a.B0, gives, warp_sum);
  __syncthreads();
  const int n_free = min(max(*a.n_free, 0), a.N);
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
  const int lane = threadIdx.x & 31;
  const int warp = blockIdx.x * WARPS + (threadIdx.x >> 5), warps = gridDim.x * WARPS;
  const int thread = blockIdx.x * THREADS + threadIdx.x, threads = gridDim.x * THREADS;
  for (int b = warp; b < a.B; b += warps) {
    const int r = row_of(b), held0 = held_before(r);
    int* row = a.table + (size_t)b * a.W;
    for (int c = lane; c < a.W; c += 32) row[c] = page_at(b, r, held0, c);
    if (lane == 0) {
      a.kv_len[b] = length_of(b) + fresh_of(b);
      a.held[b] = held0 + max(0, min(takes[b + 1], have) - min(takes[b], have));
    }
  }
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
  for (int i = thread; i < a.N; i += threads) a.free_out[i] = i < left ? pool(took + i) : -1;
  for (int b = thread; b <= a.B; b += threads) a.q_start[b] = starts[b];
  if (blockIdx.x == 0) {
    int over = 0;
    for (int b = threadIdx.x; b < a.B; b += THREADS) over += max(0, pages_of(length_of(b) + fresh_of(b), a.page_size) - a.W);
    over = __reduce_add_sync(0xffffffffu, over);
    if (lane == 0) warp_sum[threadIdx.x >> 5] = over;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < WARPS; ++w) over += warp_sum[w];
      *a.missing = takes[a.B] - took + over + max(0, left - a.N);   // (what the new list has no place for is lost)
      *a.n_free_out = min(left, a.N);
    }
  }
}

size_t smem_for(int B, int B0) { return (size_t)(2 * (B + 1) + B0 + 1 + (B0 + 31) / 32) * sizeof(int); }

}  // namespace

// Every pointer is device memory of int32, see Args; outputs overlap no input.  n_free_out, missing: one int each.
JB_EXPORT int jb_step_tables(const int* lengths, const int* fresh, const int* rows, const int* old_table, const int* old_held,
                             const int* prefix, const int* free_pages, const int* n_free, int* q_start, int* kv_len,
                             int* positions, int* token_seq, int* dest, int* table, int* held, int* free_out, int* n_free_out,
                             int* missing, int B, int B0, int T, int W0, int W, int P, int N, int page_size, cudaStream_t stream) {
  JB_REFUSE(B < 0 || B0 < 0 || T < 0 || W <= 0 || W0 < 0 || P < 0 || N < 0 || page_size <= 0, "step_tables: sizes %d %d %d %d %d %d %d %d", B, B0,
            T, W, W0, P, N, page_size);
  JB_REFUSE(W < W0 || P > W, "step_tables: a table of %d pages a row cannot take over rows of %d behind %d shared pages", W, W0, P);
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
  const Args a{lengths, fresh, rows, old_table, old_held, prefix, free_pages, n_free, q_start, kv_len, positions, token_seq, dest,
               table, held, free_out, n_free_out, missing, B, B0, T, W0, W, P, N, page_size};
  const long long work = (long long)B * W + 3ll * T + N;
  const int blocks = (int)(work / 4096 < 1 ? 1 : work / 4096 > 148 ? 148 : work / 4096);
  jb::Launch cfg(dim3(blocks), dim3(THREADS), smem, stream);
  return (int)cudaLaunchKernelEx(&cfg.c, step_tables_kernel, a);
}
