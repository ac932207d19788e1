// Page state on the device, for caches whose sequences share pages: forking
// sequences, extending them (with copy-on-write of a shared partial page),
// truncating them, and closing the gaps of a pool.
//
// State: page_refs[P], the number of table entries that hold a page (0: free);
// page_table[R][W], each sequence's pages in order, -1 past its end; kv_lens[R],
// its tokens.  A sequence of n tokens holds ceil(n / page_len) pages.  Fresh
// pages are handed out lowest first, as KvCachePool.allocate does
// (flashinfer/cache_manager.py:89-97), so the same calls give the same tables.
//
// Every result is an integer or a byte copy and independent of the order in
// which threads run: counts are summed, a page's new holder is found from its
// rank among the free pages.
#include <limits.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace pts {
namespace {

// Status bits (0: done).  Fork, extend: any bit, and nothing has changed.
constexpr int kBadIndex = 1;       // a row outside the table, or a negative count
constexpr int kTwice = 2;          // a row listed twice
constexpr int kTooLong = 4;        // a sequence longer than the table is wide
constexpr int kNoPages = 8;        // not enough free pages

constexpr int kMaxRows = 1 << 17;      // sequences of a table (a bitmap of them in shared memory)
constexpr int kMaxPoolPages = 1 << 20; // pages of a pool (a bitmap of them in shared memory)
constexpr int kMaxForks = 1024;        // forks per call
constexpr int kMaxBatch = 4096;        // sequences per extend

constexpr int kForkThreads = 256;
constexpr int kStageEntries = 8192;    // page-table entries a fork CTA holds (32 KB)

struct PageState {
  int32_t* refs;
  int32_t* table;
  int64_t stride;          // elements between table rows
  int32_t* lens;
  int rows, width, pages;
};

// One thread of a call: its status, and a failure also in the caller's word.
__device__ __forceinline__ void report(int32_t* status, int32_t* failures, int code) {
  *status = code;
  if (code && failures) atomicOr(failures, code);
}

// Marks row r in the bitmap; false if it was marked before.
__device__ __forceinline__ bool mark(uint32_t* bitmap, int r) {
  const uint32_t bit = 1u << (r & 31);
  return (atomicOr(&bitmap[r >> 5], bit) & bit) == 0;
}

// ---------------------------------------------------------------------- fork
// table[dst[i]] = table[src[i]] as it was before the call, for all i at once
// (rows may be sources and destinations, as in a beam reorder), with the pages'
// counts and the lengths.  A CTA owns `cols` columns of every row involved: it
// reads all sources' entries into shared memory, waits, then exchanges the
// destinations' entries.  Columns are independent, so no CTA waits on another.
// Bound by latency: lengths of the lists, their entries, the counts, one after the
// other (128 forks of 95 columns: 49 KB in 6.4 us from a cold cache, 6 forks 4 us); an
// entry that does not change (a child that keeps its parent's prefix) costs no atomics.
__global__ void __launch_bounds__(kForkThreads) cache_fork_kernel(PageState s, const int32_t* src, const int32_t* dst,
                                                                  int n, int cols, int32_t* status,
                                                                  int32_t* failures) {
  extern __shared__ uint32_t seen[];                    // rows listed as destinations
  __shared__ int32_t stage[kStageEntries];
  __shared__ int32_t from[kMaxForks], to[kMaxForks];
  __shared__ int bad;
  pdl_trigger();
  for (int i = threadIdx.x; i < (s.rows + 31) / 32; i += kForkThreads) seen[i] = 0u;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  pdl_wait();
  for (int i = threadIdx.x; i < n; i += kForkThreads) {
    const int a = src[i], b = dst[i];
    from[i] = a;
    to[i] = b;
    if (a < 0 || a >= s.rows || b < 0 || b >= s.rows) atomicOr(&bad, kBadIndex);
    else if (!mark(seen, b)) atomicOr(&bad, kTwice);
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) report(status, failures, bad);
  if (bad) return;
  const int c0 = blockIdx.x * cols;
  int32_t len[kMaxForks / kForkThreads];
  if (blockIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < kMaxForks / kForkThreads; ++k) {
      const int i = threadIdx.x + k * kForkThreads;
      if (i < n) len[k] = s.lens[from[i]];
    }
  }
  // entry e: column e % cols of fork e / cols; its new page waits in shared memory, the page
  // it replaces in a register (the first kHeld of a thread's entries, else read again)
  constexpr int kHeld = 4;
  int old[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    const int e = threadIdx.x + u * kForkThreads, c = c0 + e % cols;
    if (e < n * cols && c < s.width) {
      stage[e] = s.table[from[e / cols] * s.stride + c];
      old[u] = s.table[to[e / cols] * s.stride + c];
    }
  }
  for (int e = threadIdx.x + kHeld * kForkThreads; e < n * cols; e += kForkThreads)
    if (c0 + e % cols < s.width) stage[e] = s.table[from[e / cols] * s.stride + c0 + e % cols];
  __syncthreads();
  auto exchange = [&](int e, int before) {
    const int page = stage[e];
    if (page == before) return;
    s.table[to[e / cols] * s.stride + c0 + e % cols] = page;
    if (page >= 0 && page < s.pages) atomicAdd(&s.refs[page], 1);
    if (before >= 0 && before < s.pages) atomicSub(&s.refs[before], 1);
  };
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    const int e = threadIdx.x + u * kForkThreads;
    if (e < n * cols && c0 + e % cols < s.width) exchange(e, old[u]);
  }
  for (int e = threadIdx.x + kHeld * kForkThreads; e < n * cols; e += kForkThreads)
    if (c0 + e % cols < s.width) exchange(e, s.table[to[e / cols] * s.stride + c0 + e % cols]);
  if (blockIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < kMaxForks / kForkThreads; ++k) {
      const int i = threadIdx.x + k * kForkThreads;
      if (i < n) s.lens[to[i]] = len[k];
    }
  }
}

// ------------------------------------------------------------------ truncate
// One CTA per listed row: the row's length becomes min(length, new length) and
// the pages past it lose this holder.  The length and the entries are taken with
// atomics, so a row listed twice ends at the smaller length and gives each page
// back once.  Bound by latency (512 rows 4.4-5 us from a cold cache).
__global__ void __launch_bounds__(128) cache_truncate_kernel(PageState s, int page_len, const int32_t* rows,
                                                             const int32_t* new_lens, int n, int32_t* status,
                                                             int32_t* failures) {
  __shared__ int old_len;
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == gridDim.x - 1) {                    // the status: any row outside the table
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += 128) bad |= rows[i] < 0 || rows[i] >= s.rows;
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) report(status, failures, bad ? kBadIndex : 0);
    return;
  }
  const int i = blockIdx.x, r = rows[i];
  if (r < 0 || r >= s.rows) return;
  const int keep = new_lens ? max(new_lens[i], 0) : 0;
  if (threadIdx.x == 0) old_len = atomicMin(&s.lens[r], keep);
  __syncthreads();
  const int64_t end = min((int64_t)s.width, ((int64_t)old_len + page_len - 1) / page_len);
  for (int64_t j = ((int64_t)keep + page_len - 1) / page_len + threadIdx.x; j < end; j += 128) {
    const int page = atomicExch(&s.table[r * s.stride + j], -1);
    if (page >= 0 && page < s.pages) atomicSub(&s.refs[page], 1);
  }
}

// ------------------------------------------------------- bitmaps of the pool
// A plan is made by one CTA: pages of a pool are counted in tens of thousands at
// most (180 GB over some MB a page), so their counts are a few hundred KB, read
// once into a bitmap; what follows is ranks in that bitmap.
constexpr int kPlanThreads = 1024;

// bitmap bit p = (refs[p] > 0) == live, for pages from `begin` (a multiple of kRound) to
// `end`.  Four counts per load, eight loads in flight per thread; eight lanes make a word.
constexpr int kRound = 8 * 4 * kPlanThreads;            // pages that one round of loads covers

__device__ void build_bitmap(const int32_t* refs, int pages, bool live, uint32_t* bitmap, int begin, int end) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int quads = (min(pages, end) + 3) / 4;
  constexpr int kUnroll = 8;
  const bool aligned = ((uintptr_t)refs & 15) == 0;
  for (int q0 = begin / 4 + warp * 32 * kUnroll; q0 < quads; q0 += kPlanThreads * kUnroll) {
    uint32_t nib[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int q = q0 + u * 32 + lane;
      int4 v = make_int4(0, 0, 0, 0);
      int have = 0;
      if (q < quads) {
        have = min(4, pages - 4 * q);
        if (aligned && have == 4) {
          v = __ldcg(reinterpret_cast<const int4*>(refs) + q);
        } else {
          v.x = __ldcg(refs + 4 * q);
          if (have > 1) v.y = __ldcg(refs + 4 * q + 1);
          if (have > 2) v.z = __ldcg(refs + 4 * q + 2);
          if (have > 3) v.w = __ldcg(refs + 4 * q + 3);
        }
      }
      uint32_t n = ((v.x > 0) == live ? 1u : 0u) | ((v.y > 0) == live ? 2u : 0u) | ((v.z > 0) == live ? 4u : 0u) |
                   ((v.w > 0) == live ? 8u : 0u);
      nib[u] = (n & ((1u << have) - 1u)) << (4 * (lane & 7));
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      uint32_t w = nib[u];
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      w |= __shfl_xor_sync(0xffffffffu, w, 4);
      const int word = (q0 + u * 32) / 8 + (lane >> 3);
      if ((lane & 7) == 0 && word < (pages + 31) / 32) bitmap[word] = w;
    }
  }
}

// Exclusive sum over the CTA's threads of a pair of counts packed in 64 bits;
// *total receives the sums.  `part` holds 33 values.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* part,
                                                         unsigned long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();                                      // part may still be read from an earlier scan
  if (lane == 31) part[warp] = x;
  __syncthreads();
  if (warp == 0) {
    const unsigned long long w = part[lane];
    unsigned long long z = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) z += y;
    }
    part[lane] = z - w;
    if (lane == 31) part[32] = z;
  }
  __syncthreads();
  *total = part[32];
  return part[warp] + x - v;
}

// Ranks in a bitmap: thread t owns words [t * per, (t + 1) * per); below[t] set
// bits lie before them.  Returns the number of set bits.
__device__ int rank_bitmap(const uint32_t* bitmap, int words, int per, int* below, unsigned long long* part) {
  int c = 0;
  for (int w = threadIdx.x * per; w < min(words, (int)(threadIdx.x + 1) * per); ++w) c += __popc(bitmap[w]);
  unsigned long long total;
  below[threadIdx.x] = (int)block_scan((unsigned long long)c, part, &total);
  __syncthreads();
  return (int)total;
}

// The position of set bit number k (k below the number of set bits).
__device__ int select_bit(const uint32_t* bitmap, int per, const int* below, int k) {
  int t = 0;
#pragma unroll
  for (int step = kPlanThreads / 2; step > 0; step >>= 1)
    if (below[t + step] <= k) t += step;
  int left = k - below[t], w = t * per;
  for (;;) {
    const int c = __popc(bitmap[w]);
    if (left < c) break;
    left -= c;
    ++w;
  }
  uint32_t x = bitmap[w];
  int bit = 0;
#pragma unroll
  for (int half = 16; half > 0; half >>= 1) {
    const int c = __popc(x & ((1u << half) - 1u));
    if (left >= c) {
      left -= c;
      x >>= half;
      bit += half;
    }
  }
  return w * 32 + bit;
}

// -------------------------------------------------------------------- extend
struct ExtendParams {
  PageState s;
  const int32_t* rows;
  const int32_t* add_each;   // tokens per listed row, or null: `add` for every row
  int add;
  int batch;
  const int32_t* group_indptr;
  int groups;
  int page_len;
  int32_t* page_indptr;
  int32_t* page_indices;
  int32_t* last_page_len;
  int32_t* seq_lens;
  int32_t* shared_pages;     // null: not wanted
  int32_t* status;
  int32_t* failures;         // nullable
  // workspace
  int32_t* holders;          // [P] listed rows that end in this page
  int32_t* final_row;        // [P] the last of them, + 1
  int32_t* pairs;            // [batch][3]: source page, fresh page, slots
  int32_t* counts;           // pairs
  char* pool;
  int layers;
  int64_t row_bytes;
};

struct RowPlan {
  int r, old_len, need, copy, n_new;
};

// One CTA: which fresh page a row gets depends on all rows before it, and a call has few
// bytes to look at, so a scan in shared memory beats one over the GPU.  The free pages are
// a bitmap; fresh page f is its f-th set bit, found from the words' prefix sums.  Bound by
// the chain row -> length -> last page -> its count, and by the block's barriers: 6 rows
// of 2048 pages 13 us, 512 rows of 100000 pages 16 us (28 before it stopped at enough free
// pages), from a cold cache; about half of it when the state is in L2.
// kPerThread: 1 while every row has a thread of its own (the fork and extend of 6 beams
// 12.8 us in a graph; with the form that keeps 4 rows' plans per thread 14.5).
template <int kPerThread>
__global__ void __launch_bounds__(kPlanThreads) cache_extend_plan_kernel(const ExtendParams p) {
  extern __shared__ uint32_t smem[];
  const int words = (p.s.pages + 31) / 32, row_words = (p.s.rows + 31) / 32;
  uint32_t* free_bits = smem;                           // [words]
  uint32_t* seen = free_bits + words;                   // [row_words]
  int* start = (int*)(seen + row_words);                // [batch + 1] fresh pages before row i
  __shared__ int below[kPlanThreads];
  __shared__ unsigned long long part[33];
  __shared__ int bad, pairs;
  const int tid = threadIdx.x;
  pdl_trigger();
  for (int i = tid; i < row_words; i += kPlanThreads) seen[i] = 0u;
  if (tid == 0) bad = pairs = 0;
  __syncthreads();
  pdl_wait();
  const int per_row = (p.batch + kPlanThreads - 1) / kPlanThreads;      // consecutive rows of a thread
  RowPlan row[kPerThread];
  int last[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int i = tid * per_row + k;
    row[k] = RowPlan{-1, 0, 0, 0, 0};
    last[k] = -1;
    if (k >= per_row || i >= p.batch) continue;
    const int r = p.rows[i], add = p.add_each ? p.add_each[i] : p.add;
    if (r < 0 || r >= p.s.rows || add < 0) {
      atomicOr(&bad, kBadIndex);
      continue;
    }
    if (!mark(seen, r)) atomicOr(&bad, kTwice);
    const int len = p.s.lens[r];
    const long long now = (long long)len + add, most = min((long long)p.s.width * p.page_len, (long long)INT_MAX);
    if (len < 0 || len > most) {                        // not a length of this table
      atomicOr(&bad, kTooLong);
      continue;
    }
    row[k].r = r;
    row[k].old_len = len;
    row[k].n_new = (int)(((long long)len + p.page_len - 1) / p.page_len);
    if (now > most) {
      atomicOr(&bad, kTooLong);
      continue;
    }
    const int n_old = row[k].n_new;
    row[k].n_new = (int)((now + p.page_len - 1) / p.page_len);
    row[k].need = row[k].n_new - n_old;
    if (add > 0 && len % p.page_len) {
      const int page = p.s.table[r * p.s.stride + n_old - 1];
      if (page >= 0 && page < p.s.pages && __ldcg(p.s.refs + page) > 1) {
        last[k] = page;
        p.holders[page] = 0;
        p.final_row[page] = 0;
      }
    }
  }
  // the first round of counts comes in while the rows' pages are looked up
  int scanned = min(p.s.pages, kRound);
  build_bitmap(p.s.refs, p.s.pages, false, free_bits, 0, scanned);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    if (last[k] < 0) continue;
    atomicAdd(&p.holders[last[k]], 1);
    atomicMax(&p.final_row[last[k]], tid * per_row + k + 1);
  }
  __syncthreads();
  int sum = 0, lists = 0;
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    if (last[k] >= 0) {
      // the partial page stays with its last listed holder if every holder is listed
      const bool all = __ldcg(p.holders + last[k]) == __ldcg(p.s.refs + last[k]);
      row[k].copy = !(all && __ldcg(p.final_row + last[k]) == tid * per_row + k + 1);
      row[k].need += row[k].copy;
    }
    sum += row[k].need;
    lists += row[k].n_new;
  }
  unsigned long long totals;
  unsigned long long before = block_scan(((unsigned long long)(unsigned)lists << 32) | (unsigned)sum, part, &totals);
  int need_before = (int)(before & 0xffffffffu), list_before = (int)(before >> 32);
  const int want = (int)(totals & 0xffffffffu);
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int i = tid * per_row + k;
    if (k < per_row && i < p.batch) {
      start[i] = need_before;
      need_before += row[k].need;
    }
  }
  if (tid == 0) start[p.batch] = want;
  // Fresh pages are the lowest free ones, so the counts are read only until there are enough
  int per, have;
  for (;;) {
    const int w = (scanned + 31) / 32;
    per = (w + kPlanThreads - 1) / kPlanThreads;
    have = rank_bitmap(free_bits, w, per, below, part);   // synchronises: start and bad are complete
    if (have >= want || scanned >= p.s.pages) break;
    const int more = min(p.s.pages, scanned + 4 * kRound);
    build_bitmap(p.s.refs, p.s.pages, false, free_bits, scanned, more);
    scanned = more;
    __syncthreads();
  }
  int failed = bad;
  if (!failed && want > have) failed = kNoPages;
  // Unchanged, and a batch of empty sequences: an append to it writes nothing (its tokens'
  // positions would otherwise be the last ones that are there, on pages that others may hold)
  if (tid == 0) {
    report(p.status, p.failures, failed);
    p.page_indptr[0] = 0;
  }
  if (p.shared_pages)
    for (int g = tid; g < p.groups; g += kPlanThreads)
      p.shared_pages[g] = !failed && p.group_indptr[g + 1] > p.group_indptr[g] ? INT_MAX : 0;
  __syncthreads();
  // each listed row: its length and its place in the batch's lists; its shared page goes back
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int i = tid * per_row + k;
    if (k >= per_row || i >= p.batch) continue;
    const int add = p.add_each ? p.add_each[i] : p.add;
    const int now = failed ? 0 : row[k].old_len + add;
    list_before = failed ? 0 : list_before + row[k].n_new;
    p.page_indptr[i + 1] = list_before;
    p.seq_lens[i] = now;
    p.last_page_len[i] = now > 0 ? (now - 1) % p.page_len + 1 : 0;
    if (!failed) {
      p.s.lens[row[k].r] = now;
      if (row[k].copy) {
        atomicSub(&p.s.refs[last[k]], 1);
        const int fresh = select_bit(free_bits, per, below, start[i]);
        const int at = atomicAdd(&pairs, 1);            // the copies' order changes nothing
        p.pairs[3 * at] = last[k];
        p.pairs[3 * at + 1] = fresh;
        p.pairs[3 * at + 2] = row[k].old_len % p.page_len;
      }
    }
    if (!failed && p.shared_pages && p.groups > 0) {
      int lo = 0, hi = p.groups;                        // the group of row i
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.group_indptr[mid] <= i) lo = mid;
        else hi = mid;
      }
      atomicMin(&p.shared_pages[lo], row[k].old_len / p.page_len);
    }
  }
  if (failed) {
    if (tid == 0) p.counts[0] = 0;
    return;
  }
  __syncthreads();
  // fresh page number f: a row's copied page first, then its new ones, so that
  // the last of them is the row's last page
  for (int f = tid; f < want; f += kPlanThreads) {
    int lo = 0, hi = p.batch;                           // start[lo] <= f < start[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start[mid] <= f) lo = mid;
      else hi = mid;
    }
    const int page = select_bit(free_bits, per, below, f);
    const int n_pages = p.page_indptr[lo + 1] - p.page_indptr[lo];
    p.s.table[p.rows[lo] * p.s.stride + n_pages - (start[lo + 1] - f)] = page;
    p.s.refs[page] = 1;
  }
  if (tid == 0) p.counts[0] = pairs;
}

// Copies `bytes` (a multiple of 16) with kCopyThreads threads, four loads in
// flight per thread.
constexpr int kCopyThreads = 256;
__device__ __forceinline__ void copy_bytes(const char* src, char* dst, int64_t bytes) {
  const uint4* s = (const uint4*)src;
  uint4* d = (uint4*)dst;
  const int64_t n = bytes / 16;
  int64_t i = threadIdx.x;
  for (; i + 3 * kCopyThreads < n; i += 4 * kCopyThreads) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = __ldcs(s + i + u * kCopyThreads);
#pragma unroll
    for (int u = 0; u < 4; ++u) __stcs(d + i + u * kCopyThreads, v[u]);
  }
  for (; i < n; i += kCopyThreads) __stcs(d + i, __ldcs(s + i));
}

// After the plan, over all CTAs: the batch's page lists with the groups' common
// leading pages (one warp per row), and the copies of the shared partial pages
// (one CTA per page, layer and K or V).  Bound by the copies where there are any (112
// pages of 16 layers, 69 MB to be read and written: 15 us, 4.6 TB/s through L2), else by
// latency (512 rows' lists 6.6 us, 6 beams' 3 MB 5 us, both from a cold cache).
__global__ void __launch_bounds__(kCopyThreads) cache_extend_apply_kernel(const ExtendParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kWarps = kCopyThreads / 32;
  for (int i = blockIdx.x * kWarps + warp; i < p.batch; i += gridDim.x * kWarps) {
    const int r = p.rows[i];
    if (r < 0 || r >= p.s.rows) continue;               // an empty list
    const int at = p.page_indptr[i], n = p.page_indptr[i + 1] - at;
    const int32_t* mine = p.s.table + r * p.s.stride;
    int g = 0, limit = 0, head = 0;
    const int32_t* first = mine;
    if (p.shared_pages && p.groups > 0) {
      int hi = p.groups;
      while (hi - g > 1) {
        const int mid = (g + hi) >> 1;
        if (p.group_indptr[mid] <= i) g = mid;
        else hi = mid;
      }
      head = p.group_indptr[g];
      const int r0 = head >= 0 && head < p.batch ? p.rows[head] : -1;
      if (r0 >= 0 && r0 < p.s.rows) first = p.s.table + r0 * p.s.stride;
      limit = head == i ? 0 : n;                        // the first row's own list differs nowhere
    }
    int differs = INT_MAX;
    for (int j = lane; j < n; j += 32) {
      const int page = mine[j];
      p.page_indices[at + j] = page;
      if (j < limit && differs == INT_MAX && first[j] != page) differs = j;
    }
    if (limit > 0) {
      differs = __reduce_min_sync(0xffffffffu, differs);
      if (lane == 0 && differs < n) atomicMin(&p.shared_pages[g], differs);
    }
  }
  const int pairs = p.counts[0], units = pairs * p.layers * 2;
  const int64_t half = (int64_t)p.page_len * p.row_bytes;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int pair = u / (2 * p.layers), lkv = u % (2 * p.layers);
    const int from = p.pairs[3 * pair], to = p.pairs[3 * pair + 1], slots = p.pairs[3 * pair + 2];
    char* layer = p.pool + (int64_t)(lkv >> 1) * p.s.pages * 2 * half + (lkv & 1) * half;
    copy_bytes(layer + from * 2 * half, layer + to * 2 * half, slots * p.row_bytes);
  }
}

// ------------------------------------------------------------------- compact
struct CompactParams {
  PageState s;
  int page_len;
  char* pool;
  int layers;
  int64_t row_bytes;
  int32_t* out_refs;
  int32_t* out_table;        // [R][W] contiguous
  int32_t* out_map;
  int32_t* out_counts;       // live pages, moved pages
  int32_t* pairs;            // workspace [P][2]: source, destination
};

// With n live pages, the k-th live page at or past n moves to the k-th free page
// below n: no page is both a source and a destination, so the copies need no
// staging, and no copy is made that a dense pool does not need.
__global__ void __launch_bounds__(kPlanThreads) cache_compact_plan_kernel(const CompactParams p) {
  extern __shared__ uint32_t live[];
  __shared__ int below[kPlanThreads];
  __shared__ unsigned long long part[33];
  __shared__ int kept;
  const int tid = threadIdx.x, words = (p.s.pages + 31) / 32, per = (words + kPlanThreads - 1) / kPlanThreads;
  pdl_trigger();
  pdl_wait();
  if (tid == 0) kept = 0;
  build_bitmap(p.s.refs, p.s.pages, true, live, 0, p.s.pages);
  __syncthreads();
  const int n = rank_bitmap(live, words, per, below, part);
  int c = 0;                                            // live pages below n
  for (int w = tid; w * 32 < n; w += kPlanThreads) {
    const int left = n - w * 32;
    c += __popc(live[w] & (left >= 32 ? 0xffffffffu : (1u << left) - 1u));
  }
  c = __reduce_add_sync(0xffffffffu, c);
  if ((tid & 31) == 0 && c) atomicAdd(&kept, c);
  __syncthreads();
  const int stay = kept, moved = n - stay;
  for (int k = tid; k < moved; k += kPlanThreads) {
    const int from = select_bit(live, per, below, stay + k);
    p.pairs[2 * k] = from;
  }
  __syncthreads();
  for (int w = tid; w < words; w += kPlanThreads) live[w] = ~live[w];   // the free pages
  __syncthreads();
  rank_bitmap(live, words, per, below, part);
  for (int k = tid; k < moved; k += kPlanThreads) {
    const int from = p.pairs[2 * k], to = select_bit(live, per, below, k);   // holes below n come first
    p.pairs[2 * k + 1] = to;
    p.out_map[from] = to;
    p.out_refs[to] = p.s.refs[from];
  }
  if (tid == 0) {
    p.out_counts[0] = n;
    p.out_counts[1] = moved;
  }
}

// Everything but the moved pages' map: the counts, the new table, the copies.  Bound by
// HBM: 16 layers of 1.0 GB that move 354 us, 5.9 TB/s read and written.
// A CTA's share of a page copy: 16 KB pieces keep every SM supplied when few
// pages move.
constexpr int64_t kPieceBytes = 16384;

__global__ void __launch_bounds__(kCopyThreads) cache_compact_apply_kernel(const CompactParams p) {
  pdl_trigger();
  pdl_wait();
  const int n = p.out_counts[0], moved = p.out_counts[1];
  const int64_t stride = (int64_t)gridDim.x * kCopyThreads, first = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x;
  for (int64_t i = first; i < p.s.pages; i += stride) {
    const int refs = p.s.refs[i];
    if (i < n) {
      if (refs > 0) {                                   // stays (a hole's entry is the plan's)
        p.out_refs[i] = refs;
        p.out_map[i] = (int)i;
      } else {
        p.out_map[i] = -1;
      }
    } else {
      if (refs <= 0) p.out_map[i] = -1;                 // a moved page's entry is the plan's
      p.out_refs[i] = 0;
    }
  }
  for (int64_t i = first; i < (int64_t)p.s.rows * p.s.width; i += stride) {
    const int page = p.s.table[i / p.s.width * p.s.stride + i % p.s.width];
    int to = -1;
    if (page >= 0 && page < p.s.pages && p.s.refs[page] > 0) to = page < n ? page : p.out_map[page];
    p.out_table[i] = to;
  }
  const int64_t page_bytes = 2 * p.page_len * p.row_bytes;
  const int pieces = (int)((page_bytes + kPieceBytes - 1) / kPieceBytes);
  const int64_t units = (int64_t)moved * p.layers * pieces;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int piece = (int)(u % pieces);
    const int64_t pl = u / pieces, pair = pl / p.layers, l = pl % p.layers;
    char* base = p.pool + l * p.s.pages * page_bytes + piece * kPieceBytes;
    copy_bytes(base + p.pairs[2 * pair] * page_bytes, base + p.pairs[2 * pair + 1] * page_bytes,
               min(kPieceBytes, page_bytes - piece * kPieceBytes));
  }
}

int check_state(const int32_t* refs, const int32_t* table, int64_t stride, const int32_t* lens, int rows, int width,
                int pages, bool need_lens) {
  PTS_CHECK_ARG(refs && table && (lens || !need_lens), "null page state");
  PTS_CHECK_ARG(rows > 0 && width > 0 && pages > 0 && stride >= width, "bad page-table sizes");
  if (rows > kMaxRows) return set_error(PTS_ERR_CAPACITY, "%d sequences above %d", rows, kMaxRows);
  if (pages > kMaxPoolPages) return set_error(PTS_ERR_CAPACITY, "%d pages above %d", pages, kMaxPoolPages);
  return PTS_OK;
}

int check_pool(const void* pool, int layers, int page_len, int64_t row_bytes) {
  PTS_CHECK_ARG(pool && layers > 0 && page_len > 0 && row_bytes > 0, "bad pool");
  PTS_CHECK_ARG(row_bytes % 16 == 0 && ((uintptr_t)pool & 15) == 0, "rows must be whole 16-byte vectors");
  return PTS_OK;
}

int copy_grid() {
  static std::atomic<int> counts[64];                    // SMs per device
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148 * 4;
  sms = counts[dev].load();
  if (!sms) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
    counts[dev].store(sms);
  }
  return sms * 4;
}

}  // namespace
}  // namespace pts

using namespace pts;

extern "C" int pts_cache_fork(int32_t* page_refs, int32_t* page_table, int64_t table_stride, int32_t* kv_lens,
                              int num_rows, int table_width, int max_pages, const int32_t* src_rows,
                              const int32_t* dst_rows, int num_forks, int32_t* status, pts_stream_t stream) {
  return pts_cache_fork_noted(page_refs, page_table, table_stride, kv_lens, num_rows, table_width, max_pages, src_rows,
                              dst_rows, num_forks, status, nullptr, stream);
}

extern "C" int pts_cache_fork_noted(int32_t* page_refs, int32_t* page_table, int64_t table_stride, int32_t* kv_lens,
                                    int num_rows, int table_width, int max_pages, const int32_t* src_rows,
                                    const int32_t* dst_rows, int num_forks, int32_t* status, int32_t* failures,
                                    pts_stream_t stream) {
  if (int rc = check_state(page_refs, page_table, table_stride, kv_lens, num_rows, table_width, max_pages, true))
    return rc;
  PTS_CHECK_ARG(src_rows && dst_rows && status && num_forks > 0, "bad fork list");
  if (num_forks > kMaxForks) return set_error(PTS_ERR_CAPACITY, "%d forks above %d", num_forks, kMaxForks);
  const PageState s{page_refs, page_table, table_stride, kv_lens, num_rows, table_width, max_pages};
  // a CTA's columns: a line of the table for few forks, a sector of it for many (128 forks of
  // 95 columns: 18 us in three CTAs of a line, 6.4 us in twelve of a sector)
  const int cols = num_forks <= 16 ? 32 : num_forks <= 64 ? 16 : 8;
  static_assert(8 * kMaxForks <= kStageEntries, "a CTA's entries");
  const size_t smem = (size_t)(num_rows + 31) / 32 * 4;
  if (smem > 4 * 1024)
    if (int rc = ensure_smem_attr((const void*)cache_fork_kernel, smem)) return rc;
  PTS_CUDA_TRY(launch_pdl(cache_fork_kernel, dim3((table_width + cols - 1) / cols), dim3(kForkThreads), smem,
                          (cudaStream_t)stream, s, src_rows, dst_rows, num_forks, cols, status, failures));
  return launch_status("cache_fork_kernel");
}

extern "C" int pts_cache_truncate(int32_t* page_refs, int32_t* page_table, int64_t table_stride, int32_t* kv_lens,
                                  int num_rows, int table_width, int max_pages, int page_len, const int32_t* rows,
                                  const int32_t* new_lens, int num, int32_t* status, pts_stream_t stream) {
  return pts_cache_truncate_noted(page_refs, page_table, table_stride, kv_lens, num_rows, table_width, max_pages,
                                  page_len, rows, new_lens, num, status, nullptr, stream);
}

extern "C" int pts_cache_truncate_noted(int32_t* page_refs, int32_t* page_table, int64_t table_stride,
                                        int32_t* kv_lens, int num_rows, int table_width, int max_pages, int page_len,
                                        const int32_t* rows, const int32_t* new_lens, int num, int32_t* status,
                                        int32_t* failures, pts_stream_t stream) {
  if (int rc = check_state(page_refs, page_table, table_stride, kv_lens, num_rows, table_width, max_pages, true))
    return rc;
  PTS_CHECK_ARG(rows && status && num > 0 && page_len > 0, "bad row list");
  const PageState s{page_refs, page_table, table_stride, kv_lens, num_rows, table_width, max_pages};
  PTS_CUDA_TRY(launch_pdl(cache_truncate_kernel, dim3(num + 1), dim3(128), 0, (cudaStream_t)stream, s, page_len, rows,
                          new_lens, num, status, failures));
  return launch_status("cache_truncate_kernel");
}

extern "C" size_t pts_cache_workspace_size(int max_pages, int batch) {
  if (max_pages <= 0 || batch < 0) return 0;
  return ((size_t)2 * max_pages + (size_t)3 * batch + 4) * sizeof(int32_t);
}

extern "C" int pts_cache_extend(const pts_cache_extend_args* args, void* workspace, size_t workspace_bytes,
                                pts_stream_t stream) {
  return pts_cache_extend_noted(args, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int pts_cache_extend_noted(const pts_cache_extend_args* args, int32_t* failures, void* workspace,
                                      size_t workspace_bytes, pts_stream_t stream) {
  PTS_CHECK_ARG(args, "null arguments");
  const pts_cache_extend_args& x = *args;
  if (int rc = check_state(x.page_refs, x.page_table, x.table_stride, x.kv_lens, x.num_rows, x.table_width, x.max_pages, true))
    return rc;
  if (int rc = check_pool(x.kv_pool, x.num_layers, x.page_len, x.row_bytes)) return rc;
  PTS_CHECK_ARG(x.rows && x.page_indptr && x.page_indices && x.last_page_len && x.seq_lens && x.status, "null pointer");
  PTS_CHECK_ARG(x.batch > 0 && x.add >= 0 && x.num_groups >= 0, "bad sizes");
  PTS_CHECK_ARG(!x.shared_pages || (x.group_indptr && x.num_groups > 0), "shared_pages needs group_indptr");
  PTS_CHECK_ARG(x.page_indices_size >= (int64_t)x.batch * x.table_width, "page_indices holds fewer than batch * width");
  if (x.batch > kMaxBatch) return set_error(PTS_ERR_CAPACITY, "%d sequences above %d", x.batch, kMaxBatch);
  if ((int64_t)x.batch * x.table_width > INT_MAX) return set_error(PTS_ERR_CAPACITY, "page lists above 2^31 entries");
  if (!workspace || workspace_bytes < pts_cache_workspace_size(x.max_pages, x.batch))
    return set_error(PTS_ERR_CAPACITY, "workspace too small");
  PTS_CHECK_ARG(((uintptr_t)workspace & 3) == 0, "workspace must be 4-byte aligned");
  ExtendParams p{};
  p.s = PageState{x.page_refs, x.page_table, x.table_stride, x.kv_lens, x.num_rows, x.table_width, x.max_pages};
  p.rows = x.rows;
  p.add_each = x.add_each;
  p.add = x.add;
  p.batch = x.batch;
  p.group_indptr = x.group_indptr;
  p.groups = x.num_groups;
  p.page_len = x.page_len;
  p.page_indptr = x.page_indptr;
  p.page_indices = x.page_indices;
  p.last_page_len = x.last_page_len;
  p.seq_lens = x.seq_lens;
  p.shared_pages = x.shared_pages;
  p.status = x.status;
  p.failures = failures;
  p.holders = (int32_t*)workspace;
  p.final_row = p.holders + x.max_pages;
  p.pairs = p.final_row + x.max_pages;
  p.counts = p.pairs + 3 * (int64_t)x.batch;
  p.pool = (char*)x.kv_pool;
  p.layers = x.num_layers;
  p.row_bytes = x.row_bytes;
  const size_t smem = ((size_t)(x.max_pages + 31) / 32 + (x.num_rows + 31) / 32 + x.batch + 1) * 4;
  auto plan = x.batch <= kPlanThreads ? cache_extend_plan_kernel<1> : cache_extend_plan_kernel<kMaxBatch / kPlanThreads>;
  if (smem > 32 * 1024)
    if (int rc = ensure_smem_attr((const void*)plan, smem)) return rc;
  PTS_CUDA_TRY(launch_pdl(plan, dim3(1), dim3(kPlanThreads), smem, (cudaStream_t)stream, p));
  if (int rc = launch_status("cache_extend_plan_kernel")) return rc;
  const int64_t units = std::max<int64_t>((int64_t)x.batch * 2 * x.num_layers, (x.batch + 7) / 8);
  PTS_CUDA_TRY(launch_pdl(cache_extend_apply_kernel, dim3((unsigned)std::min<int64_t>(copy_grid(), units)),
                          dim3(kCopyThreads), 0, (cudaStream_t)stream, p));
  return launch_status("cache_extend_apply_kernel");
}

extern "C" int pts_cache_compact(const pts_cache_compact_args* args, void* workspace, size_t workspace_bytes,
                                 pts_stream_t stream) {
  PTS_CHECK_ARG(args, "null arguments");
  const pts_cache_compact_args& x = *args;
  if (int rc = check_state(x.page_refs, x.page_table, x.table_stride, nullptr, x.num_rows, x.table_width, x.max_pages, false))
    return rc;
  if (int rc = check_pool(x.kv_pool, x.num_layers, x.page_len, x.row_bytes)) return rc;
  PTS_CHECK_ARG(x.out_refs && x.out_table && x.out_map && x.out_counts, "null output pointer");
  PTS_CHECK_ARG(x.out_refs != x.page_refs && x.out_table != x.page_table, "the outputs must not be the inputs");
  if (!workspace || workspace_bytes < pts_cache_workspace_size(x.max_pages, 0))
    return set_error(PTS_ERR_CAPACITY, "workspace too small");
  PTS_CHECK_ARG(((uintptr_t)workspace & 3) == 0, "workspace must be 4-byte aligned");
  CompactParams p{};
  p.s = PageState{const_cast<int32_t*>(x.page_refs), const_cast<int32_t*>(x.page_table), x.table_stride, nullptr, x.num_rows,
                  x.table_width, x.max_pages};
  p.page_len = x.page_len;
  p.pool = (char*)x.kv_pool;
  p.layers = x.num_layers;
  p.row_bytes = x.row_bytes;
  p.out_refs = x.out_refs;
  p.out_table = x.out_table;
  p.out_map = x.out_map;
  p.out_counts = x.out_counts;
  p.pairs = (int32_t*)workspace;
  const size_t smem = (size_t)(x.max_pages + 31) / 32 * 4;
  if (smem > 32 * 1024)
    if (int rc = ensure_smem_attr((const void*)cache_compact_plan_kernel, smem)) return rc;
  PTS_CUDA_TRY(launch_pdl(cache_compact_plan_kernel, dim3(1), dim3(kPlanThreads), smem, (cudaStream_t)stream, p));
  if (int rc = launch_status("cache_compact_plan_kernel")) return rc;
  const int64_t pieces = (2 * x.page_len * x.row_bytes + kPieceBytes - 1) / kPieceBytes;
  const int64_t units = std::max<int64_t>((int64_t)x.max_pages * x.num_layers * pieces / 2,
                                          ((int64_t)x.num_rows * x.table_width + kCopyThreads - 1) / kCopyThreads);
  PTS_CUDA_TRY(launch_pdl(cache_compact_apply_kernel,
                          dim3((unsigned)std::min<int64_t>(2 * copy_grid(), std::max<int64_t>(units, 1))),
                          dim3(kCopyThreads), 0, (cudaStream_t)stream, p));
  return launch_status("cache_compact_apply_kernel");
}
