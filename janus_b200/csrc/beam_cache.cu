// What a step of beam search does to the cache: block tables of the beams that go on, the pages they take, share and give back
// (`fork_pages`), the copies that leaves to be made (`copy_pages`), and states of a fixed size moved from row to row (`reorder_rows`).
//
// Rows come in groups of K, the beams of a request; row k of a group goes on with what row parents[k] of the group holds.  A page is
// counted once for every row that holds it (and for holders outside the tables); whole pages are never copied.
//
// All three work in place: a thread has one column (of a group's tables, of its states) for all K rows, so that it has read what
// goes elsewhere before it writes, without a second buffer or a barrier.
#include <cooperative_groups.h>
#include <algorithm>
#include <stddef.h>
#include <stdio.h>
#include <string.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int MOST_BEAMS = 32;

// ------------------------------------------------------------ tables ------------------------------------------------------------
// One cluster, as the parts of the work need what all of the part before found: the counts of pages after every row's change (their
// atomics meet in any order: only a count's last change can be to 0), then who holds a partly filled page alone, and which
// places of the free list they take otherwise.  Pages that come back are marked in a bitmap of the cluster's first block and numbered
// from it, so that lists are the same whatever the launch looks like.
//
// Bound by a chain of waits for memory: tables and counts are a megabyte at most.  A warp has 32 columns of a group's tables, so that what a row's
// parent holds is one load more; counts go down by as many atomics at once as a group has rows.  One request of 4 beams 8.2 us, 64 of 8
// with tables of 256 pages 20.  Groups of up to 8 rows have blocks of 1,024 threads, larger ones, whose rows take the registers, 512.
constexpr int FORK_BLOCKS = 8;

struct Fork {
  const int* parents;
  const int* lengths;
  const int* table;
  const int* refs;
  const int* free_pages;
  const int* n_free;
  int* kv_len;
  int* positions;
  int* dest_rows;
  int* new_table;
  int* new_refs;
  int* new_free;
  int* new_n_free;
  int* copy_src;
  int* copy_dst;
  int* copy_rows;
  int* shared;
  int* missing;
  int R, K, W, P, F, spare, page_size;
};

// The sum over the block's threads up to this one, and over all of them in `all`.  scratch: an int a warp.
template <int WARPS>
__device__ __forceinline__ int block_scan(int v, int& all, int* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  int sums = lane < WARPS ? scratch[lane] : 0;            // (every warp adds them up for itself)
  all = __reduce_add_sync(0xffffffffu, sums);
  return __reduce_add_sync(0xffffffffu, lane < warp ? sums : 0) + v;
}

template <int KM, int FORK_THREADS>
__global__ void __cluster_dims__(FORK_BLOCKS, 1, 1) __launch_bounds__(FORK_THREADS) fork_pages_kernel(const Fork a) {
  constexpr int FORK_WARPS = FORK_THREADS / 32;
  extern __shared__ unsigned smem[];
  __shared__ int scratch[FORK_WARPS];
  __shared__ int held_of[FORK_THREADS];
  cg::cluster_group cluster = cg::this_cluster();
  const int words = (a.P + 31) / 32;
  unsigned* bits = smem;                                 // pages that come back (of the first block)
  int* ranks = reinterpret_cast<int*>(smem + words);     // ... in front of each word
  unsigned* bits0 = cluster.map_shared_rank(bits, 0);
  const int tid = threadIdx.x, lane = tid & 31, K = a.K, W = a.W, p = a.page_size;
  const int thread = cluster.block_rank() * FORK_THREADS + tid;
  constexpr int ALL = FORK_BLOCKS * FORK_THREADS;
  for (int i = tid; i < words; i += FORK_THREADS) bits[i] = 0u;
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  auto pages_of = [&](int tokens) { return tokens > 0 ? (tokens - 1) / p + 1 : 0; };
  auto counted = [&](int page) { return page >= 0 && page < a.P && page != a.spare; };
  // ---- what later parts count from ----
  const int n0 = min(max(*a.n_free, 0), a.F);
  if (a.new_refs != a.refs)
    for (int i = thread; i < a.P; i += ALL) a.new_refs[i] = a.refs[i];
  if (a.new_free != a.free_pages)
    for (int i = thread; i < a.F; i += ALL) a.new_free[i] = i < n0 ? a.free_pages[i] : -1;
  for (int r = thread; r < a.R; r += ALL) a.shared[r] = W;
  // ---- rows of the new table, but for the page that takes the next token, and the pages' counts ----
  // A warp has 32 columns of a group; lane k knows row k: which it goes on with, and how many pages the two hold.
  const int tiles = (W + 31) / 32;
  bool counts_ready = false;
  for (long long tile = thread >> 5; !counts_ready || tile < (long long)a.R * tiles; tile += ALL / 32) {
    const bool there = tile < (long long)a.R * tiles;
    const int r = there ? (int)(tile / tiles) : 0, c = there ? (int)(tile % tiles) * 32 + lane : W, row0 = r * K;
    const int parent = lane < K ? a.parents[row0 + lane] : -1, length = lane < K ? max(a.lengths[row0 + lane], 0) : 0;
    const int src = parent >= 0 && parent < K ? parent : -1;
    const int length_now = __shfl_sync(0xffffffffu, length, max(src, 0));
    const int pages_now = src >= 0 ? pages_of(length_now) : 0, pages_was = pages_of(length);
    int was[KM], now[KM];
#pragma unroll
    for (int k = 0; k < KM; ++k) was[k] = k < K && c < W ? a.table[(size_t)(row0 + k) * W + c] : -1;
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      const int from = __shfl_sync(0xffffffffu, src, k), pages = __shfl_sync(0xffffffffu, pages_now, k);
      now[k] = from < 0 && c == 0 && k < K ? a.spare : -1;
      if (from >= 0 && c < pages && c < W) now[k] = a.table[(size_t)(row0 + from) * W + c];   // (the lines are on their way already)
    }
    const unsigned goes_on = __ballot_sync(0xffffffffu, src >= 0);
    // the first column in which the rows that go on differ, and no more than the whole pages of the shortest
    bool differs = false;
    int head = 0;
    bool seen = false;
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      if ((goes_on >> k) & 1u) {
        if (!seen) head = now[k], seen = true;
        else differs = differs || now[k] != head;
      }
    }
    const unsigned where = __ballot_sync(0xffffffffu, differs && c < W);
    const int lead = __reduce_min_sync(0xffffffffu, src >= 0 ? length_now / p : W);
    if (!counts_ready) {
      cluster.sync();                                    // (the first tile's numbers are on their way meanwhile)
      counts_ready = true;
    }
    if (!there) break;
    if (lane == 0) {
      const int first = min(where ? c + __ffs(where) - 1 : W, goes_on ? lead : 0);
      if (first < W) atomicMin(&a.shared[r], first);
    }
    bool changes = false;
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      const int held = c < __shfl_sync(0xffffffffu, pages_was, k) ? was[k] : -1;
      changes = changes || now[k] != held;
    }
    if (__any_sync(0xffffffffu, changes)) {
#pragma unroll
      for (int k = 0; k < KM; ++k) {
        const int held = c < __shfl_sync(0xffffffffu, pages_was, k) ? was[k] : -1;
        if (now[k] != held && counted(now[k])) atomicAdd(&a.new_refs[now[k]], 1);
      }
      int before[KM];                                    // (all are under way before the first answer is looked at)
#pragma unroll
      for (int k = 0; k < KM; ++k) {
        const int held = c < __shfl_sync(0xffffffffu, pages_was, k) ? was[k] : -1;
        before[k] = now[k] != held && counted(held) ? atomicSub(&a.new_refs[held], 1) : 0;
      }
#pragma unroll
      for (int k = 0; k < KM; ++k)
        if (before[k] == 1) atomicOr(&bits0[was[k] >> 5], 1u << (was[k] & 31));
    }
#pragma unroll
    for (int k = 0; k < KM; ++k)
      if (k < K && c < W && (a.new_table != a.table || now[k] != was[k])) a.new_table[(size_t)(row0 + k) * W + c] = now[k];
  }
  cluster.sync();
  if (cluster.block_rank() != 0) return;
  auto source = [&](int row) {                           // the row that a row goes on with, or -1
    const int b = a.parents[row];
    return b >= 0 && b < K ? row / K * K + b : -1;
  };
  auto length_of = [&](int row) { return max(a.lengths[row], 0); };
  // ---- pages that came back, numbered ----
  int freed = 0;
  for (int i0 = 0; i0 < words; i0 += FORK_THREADS) {
    const int i = i0 + tid, n = i < words ? __popc(bits[i]) : 0;
    int all;
    const int upto = block_scan<FORK_WARPS>(n, all, scratch);
    if (i < words) ranks[i] = freed + upto - n;
    freed += all;
  }
  __syncthreads();
  auto back = [&](int i) {                               // the i-th page that came back
    int lo = 0, hi = words;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (ranks[mid] <= i) lo = mid;
      else hi = mid;
    }
    unsigned left = bits[lo];
    for (int n = i - ranks[lo]; n > 0; --n) left &= left - 1;
    return lo * 32 + __ffs(left) - 1;
  };
  const int total = n0 + freed;
  // ---- every row's page for the next token ----
  const int step = FORK_THREADS / K * K;
  int taken = 0, lacking = 0;
  for (int i0 = 0; i0 < a.R * K; i0 += step) {
    const int row = i0 + tid;
    const bool mine = tid < step && row < a.R * K;
    const int s = mine ? source(row) : -1;
    const int length = s >= 0 ? length_of(s) : 0, at = length / p, part = length % p;
    const bool fits = at < W;
    int page = s >= 0 && fits && part > 0 ? __ldcg(&a.new_table[(size_t)row * W + at]) : -1;   // (another block may have written it)
    if (page >= a.P) page = -1;
    held_of[tid] = page;
    __syncthreads();
    bool keeps = false;
    if (page >= 0) {
      const int group = tid / K * K;
      int same = 0;
      bool lowest = true;
      for (int k = 0; k < K; ++k) {
        const bool holds = held_of[group + k] == page;
        same += holds;
        if (holds && group + k < tid) lowest = false;
      }
      keeps = lowest && same == __ldcg(&a.new_refs[page]);
    }
    const bool needs = s >= 0 && fits && !keeps;
    int all;
    const int upto = block_scan<FORK_WARPS>(needs, all, scratch);    // (every count above is read before one changes below)
    const int i = total - taken - upto;
    taken += all;
    if (mine) {
      int fresh = -1;
      if (needs && i >= 0) fresh = i < n0 ? a.free_pages[i] : back(i - n0);
      if (fresh >= a.P) fresh = -1;                      // (not a page)
      const int next = keeps ? page : fresh;
      const bool copies = needs && page >= 0 && fresh >= 0;
      if (needs && page >= 0) atomicSub(&a.new_refs[page], 1);
      if (fresh >= 0) a.new_refs[fresh] = 1;
      lacking += s >= 0 && next < 0;
      if (s >= 0 && fits && (!keeps)) a.new_table[(size_t)row * W + at] = next;
      a.kv_len[row] = s >= 0 ? length + 1 : 1;
      a.positions[row] = length;
      a.dest_rows[row] = s >= 0 && next >= 0 ? next * p + part : a.spare * p;
      a.copy_src[row] = copies ? page : -1;
      a.copy_dst[row] = copies ? fresh : -1;
      a.copy_rows[row] = copies ? part : 0;
    }
    __syncthreads();
  }
  // ---- the free list ----
  const int left = max(0, total - taken), listed = min(left, a.F);
  for (int i = min(n0, listed) + tid; i < max(n0, listed); i += FORK_THREADS) a.new_free[i] = i < listed ? back(i - n0) : -1;
  int all;
  block_scan<FORK_WARPS>(lacking, all, scratch);
  if (tid == 0) {
    *a.new_n_free = listed;
    *a.missing = all + max(0, left - a.F);               // (what the list has no place for is lost)
  }
}

// Whether an output lies over an input or another output (the five that may be worked on in place may be the input itself).
bool fork_overlaps(const Fork& a) {
  const char* at[18];
  static_assert(offsetof(Fork, R) == sizeof(at), "18 tensors, the inputs first");
  memcpy(at, &a, sizeof(at));
  const size_t N = (size_t)a.R * a.K, n[18] = {N, N, N * a.W, (size_t)a.P, (size_t)a.F, 1, N, N, N, N * a.W, (size_t)a.P, (size_t)a.F, 1, N, N, N, (size_t)a.R, 1};
  const int in_place[18] = {-1, -1, -1, -1, -1, -1, 1, -1, -1, 2, 3, 4, 5, -1, -1, -1, -1, -1};
  for (int i = 6; i < 18; ++i)
    for (int j = 0; j < i; ++j)
      if (n[i] > 0 && n[j] > 0 && at[i] < at[j] + 4 * n[j] && at[j] < at[i] + 4 * n[i] && !(j == in_place[i] && at[i] == at[j])) return true;
  return false;
}

// A stretch of memory that is written.  Whether any two of n share a byte, or one with a list of `words` numbers that is read (sorts them).
// `same_twice`: the very same stretch may be there again.
struct Span {
  uintptr_t at, end;
};
bool spans_overlap(Span* spans, int n, bool same_twice, const int* const* lists, int n_lists, size_t words) {
  std::sort(spans, spans + n, [](const Span& x, const Span& y) { return x.at < y.at || (x.at == y.at && x.end < y.end); });
  for (int i = 1; i < n; ++i)
    if (spans[i].at < spans[i - 1].end && !(same_twice && spans[i].at == spans[i - 1].at && spans[i].end == spans[i - 1].end)) return true;
  for (int l = 0; l < n_lists; ++l)
    for (int i = 0; i < n; ++i)
      if ((uintptr_t)lists[l] < spans[i].end && spans[i].at < (uintptr_t)lists[l] + 4 * words) return true;
  return false;
}

template <int KM, int THREADS>
cudaError_t fork_launch(const Fork& a, cudaStream_t stream) {
  const size_t memory = (size_t)((a.P + 31) / 32) * 8;
  if (memory > 40 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(fork_pages_kernel<KM, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)memory);
    if (e != cudaSuccess) return e;
  }
  jb::Launch cfg(dim3(FORK_BLOCKS), dim3(THREADS), memory, stream);
  return cudaLaunchKernelEx(&cfg.c, fork_pages_kernel<KM, THREADS>, a);
}

// ------------------------------------------------------------ copies ------------------------------------------------------------
// Bound by bytes.  A block has one page of one tensor (or a part of it); a head's first tokens lie in one piece.  512 rows' copies in 32
// tensors, 0.9 GB to and fro, 121 us (7.5 TB/s: several beams copy the same page, which L2 serves again; a page read once, 113 us at the copy
// rate); 4 rows' in as many 3.2.
constexpr int COPY_THREADS = 256;
constexpr int MOST_TENSORS = 128;

struct CopyTensor {
  char* pages;
  int heads, row_bytes;     // of a token in a head
};
struct Copy {
  CopyTensor tensors[MOST_TENSORS];
  const int* src;
  const int* dst;
  const int* rows;
  int n_pages, page_size, parts;
};

template <typename Word>
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(const __grid_constant__ Copy a) {
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  const int item = blockIdx.x, tensor = blockIdx.y / a.parts, part = blockIdx.y % a.parts;
  const int from = a.src[item], to = a.dst[item], rows = min(a.rows[item], a.page_size);
  if (from < 0 || to < 0 || from >= a.n_pages || to >= a.n_pages || rows <= 0 || from == to) return;
  const CopyTensor t = a.tensors[tensor];
  const int per_head = t.row_bytes / (int)sizeof(Word) * a.page_size, piece = t.row_bytes / (int)sizeof(Word) * rows;
  const size_t page = (size_t)t.heads * per_head;
  const Word* in = reinterpret_cast<const Word*>(t.pages) + from * page;
  Word* out = reinterpret_cast<Word*>(t.pages) + to * page;
  const int n = t.heads * piece;
  constexpr int U = 8;
  for (int i0 = part * COPY_THREADS * U + threadIdx.x; i0 < n; i0 += a.parts * COPY_THREADS * U) {
    Word v[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * COPY_THREADS, head = i / piece;
      at[u] = head * per_head + (i - head * piece);
      if (i < n) v[u] = in[at[u]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * COPY_THREADS < n) out[at[u]] = v[u];
  }
}

// ------------------------------------------------------------ states ------------------------------------------------------------
// Bound by bytes: every state that goes elsewhere is read once for all the rows it goes to (again from the block's own cache), rows
// that stay are not touched.  40 requests of 5 beams, 12 matrices of 0.5 MB a slot: 150 us for 0.83 GB (85 % of the copy rate; what
// beams are lost makes it 0.77 to 0.87); one of 4 beams 2.9.  A thread has four columns for 4 rows, two for 8, one beyond: as much as its registers hold on the way.
constexpr int MOVE_THREADS = 256;
constexpr int MOST_MATRICES = 64;

struct Move {
  char* matrices[MOST_MATRICES];
  long long row_words[MOST_MATRICES];   // of a state, in words of the kernel's type
  const int* slots;
  const int* parents;
  int K, n_slots;
};

template <typename Word, int KM, int COLUMNS>
__global__ void __launch_bounds__(MOVE_THREADS) reorder_rows_kernel(const __grid_constant__ Move a) {
  __shared__ int from_s[KM], to_s[KM], n_s;
  jb::pdl_launch_dependents();
  jb::pdl_wait();
  const int group = blockIdx.y, matrix = blockIdx.z, K = a.K;
  if (threadIdx.x < 32) {
    const int k = threadIdx.x;
    int from = -1, to = -1;
    if (k < K) {
      const int b = a.parents[group * K + k];
      if (b >= 0 && b < K && b != k) from = a.slots[group * K + b], to = a.slots[group * K + k];
    }
    const bool moves = from >= 0 && to >= 0 && from < a.n_slots && to < a.n_slots && from != to;
    const unsigned who = __ballot_sync(0xffffffffu, moves);
    if (moves) {
      const int at = __popc(who & ((1u << k) - 1u));
      from_s[at] = from;
      to_s[at] = to;
    }
    if (k == 0) n_s = __popc(who);
  }
  __syncthreads();
  const int n = n_s;
  if (n == 0) return;
  const long long words = a.row_words[matrix];
  Word* base = reinterpret_cast<Word*>(a.matrices[matrix]);
  const long long first = (long long)blockIdx.x * MOVE_THREADS * COLUMNS + threadIdx.x;
  Word v[KM][COLUMNS];
#pragma unroll
  for (int i = 0; i < KM; ++i) {
    if (i < n) {
      const Word* row = base + from_s[i] * words;
#pragma unroll
      for (int c = 0; c < COLUMNS; ++c)
        if (first + c * MOVE_THREADS < words) v[i][c] = row[first + c * MOVE_THREADS];
    }
  }
#pragma unroll
  for (int i = 0; i < KM; ++i) {
    if (i < n) {
      Word* row = base + to_s[i] * words;
#pragma unroll
      for (int c = 0; c < COLUMNS; ++c)
        if (first + c * MOVE_THREADS < words) row[first + c * MOVE_THREADS] = v[i][c];
    }
  }
}

template <typename Word, int KM, int COLUMNS>
cudaError_t move_launch(const Move& a, int matrices, int groups, long long most_words, cudaStream_t stream) {
  const long long blocks = (most_words + MOVE_THREADS * COLUMNS - 1) / (MOVE_THREADS * COLUMNS);
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  jb::Launch cfg(dim3((unsigned)blocks, groups, matrices), dim3(MOVE_THREADS), 0, stream);
  return cudaLaunchKernelEx(&cfg.c, reorder_rows_kernel<Word, KM, COLUMNS>, a);
}

template <typename Word>
cudaError_t move_for(const Move& a, int matrices, int groups, long long most_words, cudaStream_t stream) {
  if (a.K <= 4) return move_launch<Word, 4, 4>(a, matrices, groups, most_words, stream);
  if (a.K <= 8) return move_launch<Word, 8, 2>(a, matrices, groups, most_words, stream);
  if (a.K <= 16) return move_launch<Word, 16, 1>(a, matrices, groups, most_words, stream);
  return move_launch<Word, 32, 1>(a, matrices, groups, most_words, stream);
}

}  // namespace

// given: a Fork in host memory, every pointer device memory of int32.
JB_EXPORT int jb_fork_pages(const void* given, cudaStream_t stream) {
  Fork a;
  memcpy(&a, given, sizeof(a));
  JB_REFUSE(a.R < 1 || a.K < 1 || a.K > MOST_BEAMS || a.W < 1 || a.P < 1 || a.P > 512 * 1024 || a.F < 0 || a.spare < 0 || a.spare >= a.P ||
                a.page_size < 1 || (long long)a.P * a.page_size > 0x7fffffffLL || (long long)a.R * a.K > 0x7fffffffLL / 2,
            "fork_pages: %d groups of %d rows of %d pages, %d pages of %d tokens, %d free places, spare page %d", a.R, a.K, a.W, a.P, a.page_size,
            a.F, a.spare);
  if (fork_overlaps(a)) return JB_ERR_OVERLAP;
  return (int)(a.K <= 4 ? fork_launch<4, 1024>(a, stream) : a.K <= 8 ? fork_launch<8, 1024>(a, stream)
               : a.K <= 16 ? fork_launch<16, 512>(a, stream) : fork_launch<32, 512>(a, stream));
}

// pages, heads, row_bytes: host arrays of n_tensors; src, dst, rows: device arrays of n.
JB_EXPORT int jb_copy_pages(const void* pages, const void* heads, const void* row_bytes, int n_tensors, const int* src, const int* dst,
                            const int* rows, int n, int n_pages, int page_size, cudaStream_t stream) {
  JB_REFUSE(n_tensors < 1 || n_tensors > MOST_TENSORS || n < 1 || n_pages < 1 || page_size < 1, "copy_pages: %d tensors, %d copies", n_tensors, n);
  Copy a{};
  a.src = src, a.dst = dst, a.rows = rows, a.n_pages = n_pages, a.page_size = page_size;
  uintptr_t all = 0;
  long long most = 0;
  Span spans[MOST_TENSORS];
  for (int i = 0; i < n_tensors; ++i) {
    CopyTensor& t = a.tensors[i];
    t.pages = ((char* const*)pages)[i];
    t.heads = ((const int*)heads)[i];
    t.row_bytes = ((const int*)row_bytes)[i];
    const long long bytes = (long long)t.heads * t.row_bytes * page_size;
    JB_REFUSE(t.heads < 1 || t.row_bytes < 2 || t.row_bytes % 2 || bytes > 0x7fffffffLL, "copy_pages: %d heads of %d bytes a token", t.heads,
              t.row_bytes);
    all |= (uintptr_t)t.pages | (uintptr_t)t.row_bytes;
    if (bytes > most) most = bytes;
    spans[i] = Span{(uintptr_t)t.pages, (uintptr_t)t.pages + (uintptr_t)bytes * n_pages};
  }
  const int* lists[3] = {src, dst, rows};
  if (spans_overlap(spans, n_tensors, true, lists, 3, (size_t)n)) return JB_ERR_OVERLAP;
  // A block for a whole page where that gives every multiprocessor some, else a block for each of the page's parts of eight vectors a thread.
  const long long blocks = (long long)n * n_tensors, most_parts = (most + COPY_THREADS * 128 - 1) / (COPY_THREADS * 128);
  a.parts = (int)(blocks >= 148 * 16 ? 1 : most_parts < 1 ? 1 : most_parts > 64 ? 64 : most_parts);
  JB_REFUSE((long long)n_tensors * a.parts > 65535, "copy_pages: %d tensors", n_tensors);
  jb::Launch cfg(dim3(n, n_tensors * a.parts), dim3(COPY_THREADS), 0, stream);
  if (all % 16 == 0) return (int)cudaLaunchKernelEx(&cfg.c, copy_pages_kernel<uint4>, a);
  if (all % 4 == 0) return (int)cudaLaunchKernelEx(&cfg.c, copy_pages_kernel<unsigned>, a);
  return (int)cudaLaunchKernelEx(&cfg.c, copy_pages_kernel<unsigned short>, a);
}

// matrices, numbers (float32 of a state): host arrays of n_matrices; slots, parents: device arrays [groups * K].
JB_EXPORT int jb_reorder_rows(const void* matrices, const void* numbers, int n_matrices, const int* slots, const int* parents, int groups, int K,
                              int n_slots, cudaStream_t stream) {
  JB_REFUSE(n_matrices < 1 || n_matrices > MOST_MATRICES || groups < 1 || groups > 65535 || K < 1 || K > MOST_BEAMS || n_slots < 1,
            "reorder_rows: %d matrices, %d groups of %d rows", n_matrices, groups, K);
  Move a{};
  a.slots = slots, a.parents = parents, a.K = K, a.n_slots = n_slots;
  bool wide = true;
  long long most = 0;
  Span spans[MOST_MATRICES];
  for (int i = 0; i < n_matrices; ++i) {
    a.matrices[i] = ((char* const*)matrices)[i];
    a.row_words[i] = ((const long long*)numbers)[i];
    wide &= (uintptr_t)a.matrices[i] % 16 == 0 && a.row_words[i] % 4 == 0;
    if (a.row_words[i] > most) most = a.row_words[i];
    spans[i] = Span{(uintptr_t)a.matrices[i], (uintptr_t)a.matrices[i] + 4 * (uintptr_t)a.row_words[i] * n_slots};
  }
  const int* lists[2] = {slots, parents};
  if (spans_overlap(spans, n_matrices, false, lists, 2, (size_t)groups * K)) return JB_ERR_OVERLAP;
  if (!wide) return (int)move_for<float>(a, n_matrices, groups, most, stream);
  for (int i = 0; i < n_matrices; ++i) a.row_words[i] /= 4;
  return (int)move_for<float4>(a, n_matrices, groups, most / 4, stream);
}
