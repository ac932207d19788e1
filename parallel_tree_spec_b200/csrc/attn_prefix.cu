// Tree attention for requests that share leading pages, bf16 with head_dim 64 or 128
// and pages of whole 16-token runs, on the tensor cores.  Three or four launches:
//
// plan_kernel: one CTA makes the plan (which lengths are on the device only): the column
//   sets -- each group's shared columns, each request's own -- with their rows and
//   tokens, cut into work items.
// prefix_attn_kernel: the work items, one at a time per CTA (persistent, claimed from a
//   counter): a tile of 256 query rows -- (token, query head of the KV head's group),
//   a group's requests one after the other -- a KV head and a range of 128-token blocks.
//   Shared columns are read once for all rows of a group; own columns take the tree
//   mask.  Two streams of S = Q K^T, P = e^(S - m), O += P V run in a CTA so that the
//   tensor cores compute one's products while the other's exponentials run: stream t
//   holds rows 128 t .. 128 t + 127 of the tile, or, for tiles of up to 128 rows, the same
//   rows and every second block.  tcgen05 with S and O in TMEM, P written back over S as
//   the A operand of the value product; K/V by TMA into a ring; one thread per row, so
//   the softmax needs no shuffles.  Each item leaves one part per row (fp32 O, m, l).
// own_attn_kernel, when requests have at most 16 query rows per KV head (decoding) or at
//   most 16 more than whole tiles: those rows' own columns.  So few rows fill an eighth of
//   a 128-row tensor-core tile at most, and the K/V bytes serve those rows only, so HBM is
//   the bound and mma.sync m16n8k16 on transposed products, fed by TMA through a small ring
//   per warp, is enough.  It is launched to run beside the second kernel, which is bound by
//   its arithmetic: a CTA of two warps fits an SM next to that kernel's CTA (its ring and
//   its registers are kept that small).
// join_parts_kernel: joins every row's parts and writes the output (join_tiles_kernel where
//   the own columns are work items).
//
// Scores are kept in units of log2: x = s * scale * log2(e), e^(s - m) = 2^(x - m').
#include <float.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "attn_shared.cuh"
#include "sm100.cuh"

namespace pts {
namespace {

using namespace sm100;

constexpr int kBlock = 128;               // tokens per block
constexpr int kRun = 16;                  // tokens of one value product; pages are whole runs
constexpr int kRuns = kBlock / kRun;
constexpr int kTileRows = 256;
constexpr int kThreads = 384;             // warps 0 TMA, 1 MMA, 2-3 masked values, 4-7 and 8-11 softmax
// Registers: the block is launched with 128 a thread; warps 0-3 give some back and the
// softmax warps take them.  The shares stay within the launch's total.
constexpr int kLaunchRegs = 128, kHelperRegs = 48, kSoftmaxRegs = 168;
constexpr int kBoundThreads = 512;        // the launch bound that gives 128 registers
static_assert(128 * kHelperRegs + 256 * kSoftmaxRegs <= kThreads * kLaunchRegs, "the split draws on the launch's registers");
constexpr int kMaxSplits = 32;            // block ranges of a column set
constexpr int kMaxOwnSplits = 32;         // slices of a request's own columns in own_attn_kernel
constexpr int kDirectCost = 3600;          // in tokens' time: the rounds' 3 us count 600 each
// Rows per KV head up to which own_attn_kernel takes the own columns: 64 requests of 8192
// shared and 300 own tokens take, with it and with work items, 42 and 88 us at 4 rows, 56
// and 89 at 8, 65 and 92 at 12, 71 and 93 at 16 (114 and 119 with 2048 and 1500 tokens).
// The two do not cross there: 16 rows are what a warp holds in registers, and own columns of
// 17 to 128 rows pay for mostly empty tiles.
constexpr int kFewRows = 16;
constexpr float kRescale = 8.0f;          // O is rescaled when the row max grows by more than 2^8
constexpr uint32_t kColS = 0, kColO = 256;

// K (or V) in shared memory: [8-token group][64-dim half][8 tokens][64 dims],
// 128-byte-swizzled rows.  One TMA copy brings a page's tokens (up to a block) with both
// halves, and the groups of a half lie evenly apart, as the matrix descriptors want.
// SLOTS: of the ring, each K or V of a block.
template <int D, int SLOTS = D == 128 ? 4 : 6>
struct Shape {
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kGroupBytes = kHalves * 1024;
  static constexpr uint32_t kRunBytes = 2 * kGroupBytes;
  static constexpr uint32_t kSlotBytes = kRuns * kRunBytes;     // K or V of a block; Q of a stream
  static constexpr uint32_t kQHalfBytes = 128 * 128;            // Q: [half][128 rows][64 dims]
  static constexpr int kSlots = SLOTS;
  static constexpr uint32_t kOffQ = 0;
  static constexpr uint32_t kOffRing = 2 * kSlotBytes;
  static constexpr uint32_t kOffBars = kOffRing + kSlots * kSlotBytes;
  static constexpr uint32_t kSmem = kOffBars + 512;             // barriers
  static constexpr int kPartFloats = 2 * 128 * (D + 2);         // one item's part: two streams' rows
};
static_assert(Shape<128>::kSmem <= 232448 && Shape<64>::kSmem <= 232448, "shared memory above 227 KB");

// A column set: entries 0 .. groups - 1 are the groups' shared columns, groups + b the
// own columns of request b (where they are work items).
struct __align__(16) Entry {
  int tokens;     // columns
  int prefix;     // of those, the ones that every row sees; from there on the tree mask
  int rows;       // query rows per KV head
  int tok0;       // first token of the rows
  int table;      // where its page table starts
  int first;      // first work item
  int splits;     // block ranges per (row tile, KV head)
  int pages;      // a group: its shared pages
};

struct __align__(16) Item {
  int tokens, prefix, rows, tok0;         // of the entry; rows of the tile
  int table, row0, h, own;                // row0: first row of the tile; own: takes the tree mask
  int ja, jb, pad0, pad1;                 // blocks
};

struct PlanHead {
  int total, next;          // work items; the next one that nobody has claimed
};

struct __align__(16) Bars {
  Item items[2];            // by the parity of the CTA's item count
  int index[2];             // their numbers, or -1: no more
  uint64_t item_full[2], item_free[2];
  uint64_t q_ready;         // both warpgroups: done with the last item, this one's rows stored
  uint64_t full[8], empty[8];
  uint64_t s_full[2], p_full[2][2];       // P of a stream: its first and second 64 columns
  uint64_t o_full, drain;
  uint64_t merge[2];        // two block streams: stream t's m and l are in TMEM
  uint32_t tmem;
  // masked value blocks so far: in shared memory; gone over by warps 2 and 3
  volatile int arrived, cleaned[2];
  volatile int odd[4][2];   // by item count mod 4 and warp: V held infinities or NaN in masked blocks
};
static_assert(sizeof(Bars) <= 512, "barrier block");

struct PrefixParams {
  SharedAttnParams a;
  FastDiv div_g;
  int copy_tokens;          // tokens per TMA copy: the power of two in page_len, at most a block
  int page_shift;           // log2(page_len), or -1
  float scale_log2;
  // prefix_attn_kernel takes a row's maximum before the scale, which therefore has to be
  // positive there: a negative one changes the queries' signs instead, and 0 becomes the
  // smallest normal number, 2^-126 (scores up to 2^100 count as 2^-26 at most)
  float item_scale;
  uint32_t flip;            // on two packed bf16
  int* error;
  long long wait_limit;
  // plan
  int ctas;                 // of prefix_attn_kernel
  int max_items;            // parts in the workspace
  int own_items;            // own columns are work items, but for
  int tail_rows;            // up to so many rows behind a request's last whole tile
  PlanHead* head;
  Entry* entries;
  Item* items;
  float* parts;
  // own columns in own_attn_kernel
  int own_splits;           // slices of a request's columns
  float* own_o;             // [T * Hq][own_splits][D]; tails: [batch * Hkv * kFewRows][own_splits][D]
  float2* own_ml;           // the same without D

  // Where a request's rows per KV head that own_attn_kernel takes begin (all of them, where own
  // columns are no work items); rows: none.
  __device__ __forceinline__ int tail_from(int rows) const {
    if (!own_items) return 0;
    const int from = rows / kTileRows * kTileRows;
    return rows - from <= tail_rows ? from : rows;
  }
  __device__ __forceinline__ int page_of(int tok) const { return page_shift >= 0 ? tok >> page_shift : tok / a.page_len; }
};

__device__ __forceinline__ void give_up(const PrefixParams& p, int code) {
  if (p.error) atomicExch(p.error, code);
}

__device__ __forceinline__ int blocks_of(int tokens) { return (tokens + kBlock - 1) / kBlock; }
__device__ __forceinline__ int tiles_of(int rows) { return (rows + kTileRows - 1) / kTileRows; }

// a / b for 0 <= a < 2^24, 0 < b < 2^24 (the quotient by floats is off by one at most):
// the planning is a chain of these, and the compiler's integer division is a longer one.
__device__ __forceinline__ int small_div(int a, int b) {
  const int q = (int)__fdividef((float)a, (float)b), r = a - q * b;
  return q + (r >= b ? 1 : 0) - (r < 0 ? 1 : 0);
}
__device__ __forceinline__ int ceil_div(int a, int b) { return small_div(a + b - 1, b); }

__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull; }

// Which of columns c0 .. c0 + 63 row `node` (token tok of the queries) sees (bit i: column
// c0 + i): those before `prefix`, then tree slots by the row's mask, or up to its own
// without masks; none from `len` on.
__device__ __noinline__ uint64_t seen_columns(const SharedAttnParams& a, int tok, int node, int c0, int prefix,
                                              int len) {
  uint64_t v = low_bits(min(prefix, len) - c0);
  const int first = max(prefix, c0), end = min(len, c0 + 64);   // tree columns of the 64
  if (first < end) {
    const int slot = first - prefix;
    uint64_t bits;
    if (!a.mask_bits) {
      bits = low_bits(node - slot + 1);
    } else {
      const uint64_t* mask = a.mask_bits + (int64_t)tok * a.mask_words;
      const int w = slot >> 6, sh = slot & 63;
      const uint64_t lo = w < a.mask_words ? __ldg(mask + w) : 0ull;
      const uint64_t hi = sh && w + 1 < a.mask_words ? __ldg(mask + w + 1) : 0ull;
      bits = sh ? (lo >> sh) | (hi << (64 - sh)) : lo;
    }
    v |= (bits & low_bits(end - first)) << (first - c0);
  }
  return v;
}

// One of two packed bf16 values is infinite or NaN.
__device__ __forceinline__ bool odd2(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// ------------------------------------------------------------------------- plan
constexpr int kPlanThreads = 256;
constexpr int kOwnWarps = 2, kDirectWarps = 8;
constexpr int kOwnStages = 2;
constexpr int kPlanCache = 512;           // entries that the plan keeps in shared memory

// What an item costs besides its blocks, in half block times: its start and the storing of
// its part, some three blocks, and the part's share of the join.  Over 34 mixed calls (10 to
// 400 us) the geometric mean was, with 3, 9, 12, 16, 20 and 28: 53.6, 51.9, 51.5, 51.4, 51.4
// and 52.0 us (others: 46.4, 45.3, 45.1, 45.0, 45.0, 45.3), single calls up to a third less.
// One constant for shared ranges and own tiles, which would each like another: own columns of
// 4 and 8 rows as work items (which no call has) took 63 and 76 us with 3, 88 and 89 with 16.
constexpr int kItemCost = 16;

// The plan.  The launch costs about the larger of all items over the CTAs and of the large
// items' rounds; the cheapest of up to 32 ranges of ceil(longest / k) blocks is taken.  Bound by the chain
// of its loads and barriers: 4-6 us with its inputs in L2, from a cold cache 7 for 16
// requests and 8-9 for 64.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PrefixParams p) {
  __shared__ int sums[64 + 4];                          // [2][32] items, large items; red
  __shared__ Entry cache[kPlanCache];                   // the first entries, as in p.entries
  const SharedAttnParams& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int warps = kPlanThreads / 32, threads = kPlanThreads;
  pdl_wait();
  pdl_trigger();
  int* red = sums + 64;                                 // longest, blocks, chunk, total
  Entry* entry = a.groups + (p.own_items ? a.batch : 0) <= kPlanCache ? cache : p.entries;
  if (tid < 68) sums[tid] = 0;
  for (int g = warp; g < a.groups; g += warps) {
    int lead;
    const int pages = group_shared_pages(a, g, &lead);
    const int2 range = group_requests(a, g);
    const int tok0 = a.qo_indptr[range.x], rows = (a.qo_indptr[range.y] - tok0) * a.g;
    if (lane == 0) {
      const int tokens = rows > 0 ? pages * a.page_len : 0;
      entry[g] = Entry{tokens, tokens, rows, tok0, rows > 0 ? a.page_indptr[lead] : 0, 0, 0, rows > 0 ? pages : 0};
    }
  }
  __syncthreads();
  const int entries = a.groups + (p.own_items ? a.batch : 0);
  if (p.own_items) {
    for (int b = tid; b < a.batch; b += threads) {
      const int tok0 = a.qo_indptr[b], n = a.qo_indptr[b + 1] - tok0, pages = entry[group_of(a, b)].pages;
      const int len = n > 0 ? max(0, kv_tokens(a, b) - pages * a.page_len) : 0;
      entry[a.groups + b] = Entry{len, len - n, p.tail_from(n * a.g), tok0, a.page_indptr[b] + pages, 0, 0, 0};
    }
    __syncthreads();
  }
  auto shape_of = [&](int e) -> int2 {
    return make_int2(tiles_of(entry[e].rows) * a.Hkv, blocks_of(entry[e].tokens));
  };
  int longest = 1, blocks = 0;
  for (int e = tid; e < entries; e += threads) {
    const int2 x = shape_of(e);
    longest = max(longest, x.x ? x.y : 0);
    blocks += x.x * x.y;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  blocks = __reduce_add_sync(0xffffffffu, blocks);
  if (lane == 0) {
    atomicMax(&red[0], longest);
    atomicAdd(&red[1], blocks);
  }
  __syncthreads();
  longest = red[0];
  blocks = red[1];
  {
    // lane k: ranges of c blocks; each warp takes every warps-th entry
    const int c = ceil_div(longest, lane + 1);
    int items = 0, large = 0;
#pragma unroll 2
    for (int e = warp; e < entries; e += warps) {
      const int2 x = shape_of(e);
      const int full = small_div(x.y, c), rest = x.y - full * c;
      items += x.x * (full + (rest > 0));
      large += x.x * (full + (2 * rest >= c && rest > 0));
    }
    atomicAdd(&sums[lane], items);
    atomicAdd(&sums[32 + lane], large);
  }
  __syncthreads();
  if (warp == 0) {
    const int c = ceil_div(longest, lane + 1), items = sums[lane], large = sums[32 + lane];
    unsigned cost = 0xffffffffu;
    if (lane == 0 || (lane < longest && items <= p.max_items))
      cost = (unsigned)max(small_div(min(2 * blocks + kItemCost * items, (1 << 24) - 1), p.ctas),
                           small_div(min(large, 1 << 20) + p.ctas - 1, p.ctas) * (2 * c + kItemCost));
    const unsigned win = __reduce_min_sync(0xffffffffu, cost);
    const int chunk = __reduce_max_sync(0xffffffffu, cost == win ? c : 0);   // equal costs: fewer parts
    if (lane == 0) red[2] = chunk;
  }
  __syncthreads();
  const int chunk = red[2];
  // the entries' first items, warp 0 over all entries in order
  if (warp == 0) {
    int run = 0;
    for (int e0 = 0; e0 < entries; e0 += 32) {
      const int e = e0 + lane;
      int n = 0, splits = 0;
      if (e < entries) {
        const int2 x = shape_of(e);
        splits = ceil_div(x.y, chunk);
        n = x.x * splits;
      }
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (e < entries) {
        entry[e].splits = splits;
        entry[e].first = run + incl - n;
      }
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      red[3] = min(run, p.max_items);
      *p.head = PlanHead{min(run, p.max_items), p.ctas};
    }
  }
  __syncthreads();
  const int total = red[3];
  if (entry != p.entries)
    for (int e = tid; e < entries; e += threads) p.entries[e] = entry[e];
  for (int i = tid; i < total; i += threads) {
    int lo = 0, hi = entries;                           // the last entry whose first item is <= i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (entry[mid].first <= i) lo = mid;
      else hi = mid;
    }
    const Entry x = entry[lo];
    const int u = small_div(i - x.first, x.splits), split = i - x.first - u * x.splits, tiles = tiles_of(x.rows);
    const int h = small_div(u, tiles), row0 = (u - h * tiles) * kTileRows;
    p.items[i] = Item{x.tokens, x.prefix, min(kTileRows, x.rows - row0), x.tok0, x.table, row0, h, lo >= a.groups,
                      split * chunk, min(blocks_of(x.tokens), (split + 1) * chunk), 0, 0};
  }
}

// ------------------------------------------------------------------ own columns
// The own columns of a request with at most 8 NR rows.  The CTA's NW warps take its
// 16-token runs in turn, each through a ring of its own, and compute
//   S^T = K Q^T (16 tokens x 8 rows per product), O^T += V^T P^T,
// P^T handed to the second product by movmatrix; the warps' O, m and l are added up at
// the end.  Transposed, a product's 16 rows are tokens or dimensions, all of them
// in use, and the 8 columns are query rows: half the products of the plain form at 8
// rows or fewer.
// 64 requests with 225 own tokens on average, 8 KV heads of 128 (59 MB): 19 us by itself,
// 3.1 TB/s -- a pair's 14 runs are over before the ring has paid for its start -- and, two
// CTAs beside prefix_attn_kernel's on an SM, about as long as that kernel (one: 35 us
// beside its 25).
// kDirect: all columns, the shared ones too, and the output itself: for small calls, where
// reading a short prefix once per request costs less than the plan and the join.
template <int D, int NR, int NW, bool kDirect>
__global__ void __launch_bounds__(32 * NW, kDirect ? 1 : 7)
    own_attn_kernel(const PrefixParams p, const __grid_constant__ CUtensorMap run_map) {
  using S = Shape<D>;
  constexpr int kRows = 8 * NR;
  constexpr uint32_t kStage = 2 * S::kRunBytes, kWarp = kOwnStages * kStage;
  extern __shared__ __align__(1024) uint8_t smem[];      // the warps' rings; barriers behind
  constexpr int warps = NW;
  uint64_t(*full)[kOwnStages] = (uint64_t(*)[kOwnStages])(smem + warps * kWarp);
  // after the loop the rings hold the warps' O, [warps][kRows][D + 4], and (m, l)
  constexpr int kStride = D + 4;
  float2(*ml)[kRows] = (float2(*)[kRows])(smem + warps * kRows * kStride * 4);
  const SharedAttnParams& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  if (lane < kOwnStages) mbar_init(&full[warp][lane], 1);
  fence_mbar_init();
  __syncwarp();
  if (kDirect) pdl_wait();
  pdl_trigger();
  // Beside the others nothing here depends on the two kernels before: what this one reads is not theirs, and
  // everything before them had completed when they were launched.  Only the grid's last CTA
  // waits for them, so that what follows may wait for this kernel alone while the other
  // CTAs make room.
  const bool last = !kDirect && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1;
  const int b = blockIdx.x, h = blockIdx.y;
  const int tok0 = a.qo_indptr[b], n_tok = a.qo_indptr[b + 1] - tok0, total_rows = n_tok * a.g;
  const int from = kDirect || total_rows <= 0 ? 0 : p.tail_from(total_rows);
  if (total_rows <= from) {
    if (last) pdl_wait();
    return;
  }
  const int rows = min(kRows, total_rows - from);
  const int shared = kDirect ? 0 : group_shared_pages(a, group_of(a, b));
  const int32_t* table = a.page_indices + a.page_indptr[b] + shared;
  const int len = max(0, kv_tokens(a, b) - shared * a.page_len), prefix = len - n_tok;
  const int n_runs = (len + kRun - 1) / kRun;
  const int r0 = (int)((int64_t)n_runs * blockIdx.z / p.own_splits);
  const int r1 = (int)((int64_t)n_runs * (blockIdx.z + 1) / p.own_splits);
  const int mine = max(0, (r1 - r0 - warp + warps - 1) / warps);   // this warp's runs r0 + warp + warps i
  const uint32_t ring = smem_u32(smem) + warp * kWarp;

  // the pages of this warp's runs 32 w .. 32 w + 31, one per lane
  auto window = [&](int w) -> int {
    const int tok = (r0 + warp + warps * (32 * w + lane)) * kRun;
    const int page = 32 * w + lane < mine ? __ldg(table + p.page_of(tok)) : -1;
    return page >= 0 && page < a.max_pages ? page : a.max_pages;     // past the pool: zero fill
  };
  int page_now = window(0), page_next = mine > 32 ? window(1) : 0;
  auto load = [&](int i) {
    if ((i & 31) == 0 && i > 0) {
      page_now = page_next;
      page_next = i + 32 < mine ? window((i >> 5) + 1) : 0;
    }
    const int page = __shfl_sync(0xffffffffu, page_now, i & 31);
    if (lane == 0) {
      const int tok = (r0 + warp + warps * i) * kRun, group = (tok - p.page_of(tok) * a.page_len) / 8;
      uint64_t* bar = &full[warp][i % kOwnStages];
      uint8_t* dst = smem + warp * kWarp + (i % kOwnStages) * kStage;
      mbar_arrive_expect_tx(bar, kStage);
      tma_load_5d(dst, &run_map, bar, 0, 0, h * S::kHalves, group, 2 * page);
      tma_load_5d(dst + S::kRunBytes, &run_map, bar, 0, 0, h * S::kHalves, group, 2 * page + 1);
    }
    __syncwarp();
  };
  int loaded = 0;
  for (; loaded < min(kOwnStages, mine); ++loaded) load(loaded);

  // Q^T as the B operand: column gq of tile n is row 8 n + gq; rows past the request's are 0
  uint32_t qb[NR][D / 16][2];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = 8 * n + gq, R = from + r, tk = p.div_g.div(R);
    const bool valid = r < rows;
    const uint16_t* q =
        (const uint16_t*)a.q + ((int64_t)(tok0 + (valid ? tk : 0)) * a.Hq + h * a.g + (valid ? R - tk * a.g : 0)) * D + 2 * tq;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qb[n][k][0] = valid ? __ldg((const uint32_t*)(q + 16 * k)) : 0u;
      qb[n][k][1] = valid ? __ldg((const uint32_t*)(q + 16 * k + 8)) : 0u;
    }
  }
  // this lane's softmax rows: 8 n + 2 tq + {0, 1}
  float o[NR][D / 16][4], m[NR][2], l[NR][2];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.0f;
  }
  const int mi = lane >> 3, rr = lane & 7;
  bool ok = true;
  int i = 0;
  for (; i < mine; ++i) {
    const uint32_t kb = ring + (i % kOwnStages) * kStage, vb = kb + S::kRunBytes;
    ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][i % kOwnStages], (i / kOwnStages) & 1, p.wait_limit));
    if (!ok) break;
    const int c0 = (r0 + warp + warps * i) * kRun;      // own column of the run's first token
    float s[NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      uint32_t x[4];                                    // K: tokens 8 (mi & 1) + rr, dims 16 k + 8 (mi >> 1)
      const int ch = 2 * k + (mi >> 1);
      ldmatrix_x4(kb + (mi & 1) * S::kGroupBytes + (ch >> 3) * 1024 + rr * 128 + (((ch & 7) ^ rr) << 4), x[0], x[1], x[2],
                  x[3]);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma_m16n8k16(s[n], x, qb[n][k][0], qb[n][k][1]);
    }
    // element e: token gq + 8 (e >> 1), row 2 tq + (e & 1)
    const bool masked = c0 + kRun > prefix;             // tree slots or the end in this run
    bool grow = false;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      uint32_t seen[2] = {0xffffu, 0xffffu};
      if (masked) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = 8 * n + 2 * tq + j, node = p.div_g.div(from + r);
          seen[j] = r < rows ? (uint32_t)seen_columns(a, tok0 + node, node, c0, prefix, len) : 0u;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool see = (seen[e & 1] >> (gq + 8 * (e >> 1))) & 1u;
        s[n][e] = see ? s[n][e] * p.scale_log2 : -INFINITY;
        grow |= s[n][e] > m[n][e & 1] + kRescale;
      }
    }
    // the subtracted max moves only when some score exceeds it by more than 2^8
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = fmaxf(s[n][j], s[n][2 + j]);
#pragma unroll
          for (int off = 4; off <= 16; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          const float nm = fmaxf(m[n][j], top);
          const float f = nm == -INFINITY ? 1.0f : fast_exp2(m[n][j] - nm);
          m[n][j] = nm;
          l[n][j] *= f;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            o[n][d][j] *= f;
            o[n][d][2 + j] *= f;
          }
        }
    }
    uint32_t pb[NR][2];
    float e[NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float base = m[n][k & 1] == -INFINITY ? 0.0f : m[n][k & 1];
        e[n][k] = fast_exp2(s[n][k] - base);
        l[n][k & 1] += e[n][k];
      }
      pb[n][0] = movmatrix_trans(pack_bf16x2(e[n][0], e[n][1]));
      pb[n][1] = movmatrix_trans(pack_bf16x2(e[n][2], e[n][3]));
    }
    // Values in places that no row sees, or that only some rows see, may be infinite or NaN,
    // which 0 * v does not cancel: slots from the length on are zeroed, and a run that
    // holds such values is added up value by value.
    bool odd = false;
    if (masked) {
      for (int x = lane; x < kRun * D / 8; x += 32) {
        const int tok = x / (D / 8), ch = x % (D / 8);
        const uint32_t at = vb + (tok >> 3) * S::kGroupBytes + (ch >> 3) * 1024 + (tok & 7) * 128 + (((ch & 7) ^ (tok & 7)) << 4);
        if (c0 + tok >= len) {
          st_shared_v4(at, 0u, 0u, 0u, 0u);
        } else {
          const uint4 v = ld_shared_v4(at);
          odd |= odd2(v.x) || odd2(v.y) || odd2(v.z) || odd2(v.w);
        }
      }
      odd = __any_sync(0xffffffffu, odd) && (n_tok > 1 || a.mask_bits);   // (a lone causal row sees all)
      __syncwarp();
    }
    if (!odd) {
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t x[4];                                  // V^T: dims 16 d + 8 (mi & 1), tokens 8 (mi >> 1) + rr
        const int ch = 2 * d + (mi & 1);
        ldmatrix_x4_trans(vb + (mi >> 1) * S::kGroupBytes + (ch >> 3) * 1024 + rr * 128 + (((ch & 7) ^ rr) << 4), x[0],
                          x[1], x[2], x[3]);
#pragma unroll
        for (int n = 0; n < NR; ++n) mma_m16n8k16(o[n][d], x, pb[n][0], pb[n][1]);
      }
    } else {
      for (int u = 0; u < kRun; ++u) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const int from = (u & 7) * 4 + tq;
          const float p0 = __shfl_sync(0xffffffffu, u < 8 ? e[n][0] : e[n][2], from);
          const float p1 = __shfl_sync(0xffffffffu, u < 8 ? e[n][1] : e[n][3], from);
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int half = 0; half < 2; ++half) {      // dim 16 d + gq + 8 half
              const int ch = 2 * d + half;
              uint16_t w;
              asm volatile("ld.shared.u16 %0, [%1];"
                           : "=h"(w)
                           : "r"(vb + (u >> 3) * S::kGroupBytes + (ch >> 3) * 1024 + (u & 7) * 128 +
                                 (((ch & 7) ^ (u & 7)) << 4) + 2 * gq));
              const float v = bf16_bits_to_float(w);
              if (p0 != 0.0f) o[n][d][2 * half] = fmaf(p0, v, o[n][d][2 * half]);
              if (p1 != 0.0f) o[n][d][2 * half + 1] = fmaf(p1, v, o[n][d][2 * half + 1]);
            }
        }
      }
    }
    __syncwarp();
    if (loaded < mine) load(loaded++);
  }
  if (!ok) {
    if (lane == 0) give_up(p, 81);
    for (int x = i; x < loaded; ++x) mbar_wait(&full[warp][x % kOwnStages], (x / kOwnStages) & 1);
  }
  __syncthreads();
  float* os = (float*)smem;
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float sum = l[n][j];
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      const int r = 8 * n + 2 * tq + j;
      if (gq == 0) ml[warp][r] = make_float2(m[n][j], sum);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        os[(warp * kRows + r) * kStride + 16 * d + gq] = o[n][d][j];
        os[(warp * kRows + r) * kStride + 16 * d + gq + 8] = o[n][d][2 + j];
      }
    }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * (D / 4); e += blockDim.x) {
    const int r = e / (D / 4), quad = e % (D / 4), tk = p.div_g.div(from + r);
    float M = -INFINITY;
    for (int w = 0; w < warps; ++w) M = fmaxf(M, ml[w][r].x);
    const float base = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int w = 0; w < warps; ++w) {
      const float f = fast_exp2(ml[w][r].x - base);
      const float4 v = *(const float4*)(os + (w * kRows + r) * kStride + quad * 4);
      L = fmaf(f, ml[w][r].y, L);
      acc.x = fmaf(f, v.x, acc.x);
      acc.y = fmaf(f, v.y, acc.y);
      acc.z = fmaf(f, v.z, acc.z);
      acc.w = fmaf(f, v.w, acc.w);
    }
    const int64_t row = (int64_t)(tok0 + tk) * a.Hq + h * a.g + from + r - tk * a.g;
    if (kDirect) {
      const float f = L > 0.0f ? 1.0f / L : L == L ? 0.0f : L;    // nothing seen: 0
      *(uint2*)((uint16_t*)a.out + row * D + quad * 4) =
          make_uint2(pack_bf16x2(acc.x * f, acc.y * f), pack_bf16x2(acc.z * f, acc.w * f));
      continue;
    }
    const int64_t part = (p.own_items ? ((int64_t)b * a.Hkv + h) * kFewRows + r : row) * p.own_splits + blockIdx.z;
    *(float4*)(p.own_o + part * D + quad * 4) = acc;
    if (quad == 0) p.own_ml[part] = make_float2(M, L);
  }
  if (last) pdl_wait();
}

// Shared memory of own_attn_kernel: the rings (later the warps' O, m and l), barriers.
template <int D, int NR, int NW>
constexpr size_t own_smem() {
  constexpr size_t ring = (size_t)kOwnStages * 2 * Shape<D>::kRunBytes, o = (size_t)8 * NR * ((D + 4) * 4 + 8);
  static_assert(ring >= o, "the rings hold the warps' O, m and l");
  return NW * (ring + 8 * kOwnStages);
}
// with prefix_attn_kernel's CTA beside it, and two with the narrow one (each in 128 bytes
// and 1 KB more that the system takes)
constexpr size_t sm_share(size_t smem) { return (smem + 127) / 128 * 128 + 1024; }
static_assert(sm_share(own_smem<128, 2, kOwnWarps>()) + sm_share(Shape<128>::kSmem) <= 228 * 1024 &&
                  2 * sm_share(own_smem<128, 2, kOwnWarps>()) + sm_share(Shape<128, 3>::kSmem) <= 228 * 1024,
              "they fit an SM");

// ------------------------------------------------------------------- work items
// Ring positions of block i's K and V among n blocks, in load order.  Two row tiles use
// every block at once: K0 V0 K1 V1 ..; two block streams start with both streams' keys:
// K0 K1 V0 K2 V1 K3 ..
__device__ __forceinline__ int ring_k(bool two, int i) { return two ? 2 * i : i < 2 ? i : 2 * i - 1; }
__device__ __forceinline__ int ring_v(bool two, int i, int n) { return two ? 2 * i + 1 : i < n - 1 ? 2 * i + 2 : 2 * n - 1; }

// Block j of an own item holds columns that some rows do not see.
__device__ __forceinline__ bool masked_block(const Item& it, int j) {
  return it.own && (it.ja + j + 1) * kBlock > it.prefix;
}

// Bound by the chain of a stream's block: scores from TMEM, their maximum, the exponentials,
// P to TMEM, the two products.  128 tokens of 256 rows of head_dim 128 take 2.2 us (7.6
// TFLOP/s of an SM; all of them 68 % of the measured matrix rate), of which the products
// alone are 2048 clocks and the exponentials as many.  An item costs 5-9 us more for its
// start and its parts.  16 requests of up to 65 nodes with 4096 shared tokens: 80-85 us,
// the matrix pipe 35 % busy over the launch; 32 decoding requests with 65536 shared tokens:
// the cache at 5.2 TB/s.
template <int D, int SLOTS>
__global__ void __launch_bounds__(kBoundThreads, 1)
    prefix_attn_kernel(const PrefixParams p, const __grid_constant__ CUtensorMap kv_map) {
  using S = Shape<D, SLOTS>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars& bars = *reinterpret_cast<Bars*>(smem + S::kOffBars);
  const SharedAttnParams& a = p.a;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  pdl_trigger();                                        // own_attn_kernel may start beside this one

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.item_full[t], 1);
      mbar_init(&bars.item_free[t], 11);                // 8 softmax warps, 2 value warps, the MMA thread
      mbar_init(&bars.s_full[t], 1);
      mbar_init(&bars.p_full[t][0], 4);
      mbar_init(&bars.p_full[t][1], 4);
      mbar_init(&bars.merge[t], 4);
    }
    mbar_init(&bars.q_ready, 8);
    for (int s = 0; s < S::kSlots; ++s) {
      mbar_init(&bars.full[s], 1);
      mbar_init(&bars.empty[s], 1);
    }
    mbar_init(&bars.o_full, 1);
    mbar_init(&bars.drain, 1);
    bars.arrived = bars.cleaned[0] = bars.cleaned[1] = 0;
    fence_mbar_init();
    tma_prefetch_desc(&kv_map);
  }
  if (warp == 1) {
    tmem_alloc(&bars.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;

  // Item number k of this CTA, for the warps that do not hand it out: waits until it is
  // there and copies it; false when there are no more (or the wait ran out).
  auto next_item = [&](int k, Item& it) -> bool {
    if (!mbar_wait(&bars.item_full[k & 1], (k >> 1) & 1, p.wait_limit)) {
      give_up(p, 41);
      return false;
    }
    const int i = bars.index[k & 1];
    it = bars.items[k & 1];
    return i >= 0;
  };

  if (warp >= 4) {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = (warp - 4) >> 2, quarter = warp & 3;
    const int r_local = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tm = tmem + lane_base + kColS + 128 * t, o_tm = tmem + lane_base + kColO + D * t;
    bool ok = true;
    int steps = 0, merges = 0;
    // The first round is a rehearsal, while the plan is made: one pass of the block
    // code over whatever the TMEM holds, with nothing waited for, signalled or kept.
    // It brings the loop's instructions (some 10 KB) into the SM's caches, which cost the
    // first real block about 3500 cycles otherwise.
    Item it;
    it.rows = it.tokens = it.ja = it.row0 = it.h = it.tok0 = it.prefix = it.own = 0;
    it.jb = 1;
    for (int k = -1;; ++k) {
      const bool rehearse = k < 0;
      int index = 0;
      if (!rehearse) {
        ok = __all_sync(0xffffffffu, next_item(k, it));
        if (!ok) break;
        index = bars.index[k & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.item_free[k & 1]);
      }
      const bool two = it.rows > 128;
      const int n = it.jb - it.ja, count = two ? n : (n + 1 - t) / 2;
      const int my0 = two ? 128 * t : 0;                // this stream's first row of the tile
      if (!rehearse) {
        if (two || t == 0) {
          // the warp's 32 query rows into the swizzled A operand, two (D = 128) or four
          // rows per load instruction; the previous item's products have all completed
          constexpr int kChunks = D / 8, kPer = 32 / kChunks, kLoads = 32 / kPer;
          const int chunk = lane % kChunks;
          const uint32_t qb = smem_u32(smem + S::kOffQ + (two ? t : 0) * S::kSlotBytes) + (chunk / 8) * S::kQHalfBytes;
          const uint16_t* q = (const uint16_t*)a.q + ((int64_t)it.tok0 * a.Hq + it.h * a.g) * D + chunk * 8;
          uint4 v[kLoads];
#pragma unroll
          for (int j = 0; j < kLoads; ++j) {
            const int r = quarter * 32 + j * kPer + lane / kChunks, R = it.row0 + my0 + r;
            const int tk = p.div_g.div(R);
            v[j] = make_uint4(0, 0, 0, 0);
            if (my0 + r < it.rows) v[j] = __ldg((const uint4*)(q + ((int64_t)tk * a.Hq + (R - tk * a.g)) * D));
            v[j] = make_uint4(v[j].x ^ p.flip, v[j].y ^ p.flip, v[j].z ^ p.flip, v[j].w ^ p.flip);
          }
#pragma unroll
          for (int j = 0; j < kLoads; ++j) {
            const int r = quarter * 32 + j * kPer + lane / kChunks;
            st_shared_v4(qb + (uint32_t)r * 128u + (uint32_t)(((chunk & 7) ^ (r & 7)) << 4), v[j].x, v[j].y, v[j].z,
                         v[j].w);
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_ready);
      }
      const bool valid = my0 + r_local < it.rows;
      const int node = p.div_g.div(it.row0 + my0 + r_local);
      float m = -INFINITY, l = 0.0f;
      for (int x = 0; x < count; ++x) {
        if (!rehearse) {
          ok = __all_sync(0xffffffffu, mbar_wait(&bars.s_full[t], steps & 1, p.wait_limit));
          if (!ok) break;
          tc_fence_after();
        }
        uint32_t s[2][64];
        tmem_ld32_x2(s_tm, s[0]);
        tmem_ld32_x2(s_tm + 64, s[1]);
        tmem_ld_wait();
        const int c0 = (it.ja + (two ? x : 2 * x + t)) * kBlock;
        if (c0 + kBlock > it.prefix) {
          uint32_t seen[4] = {0u, 0u, 0u, 0u};
          if (valid) {
            const uint64_t lo = seen_columns(a, it.tok0 + node, node, c0, it.prefix, it.tokens);
            const uint64_t hi = seen_columns(a, it.tok0 + node, node, c0 + 64, it.prefix, it.tokens);
            seen[0] = (uint32_t)lo;
            seen[1] = (uint32_t)(lo >> 32);
            seen[2] = (uint32_t)hi;
            seen[3] = (uint32_t)(hi >> 32);
          }
#pragma unroll
          for (int c = 0; c < kBlock; ++c)
            if (!((seen[c / 32] >> (c % 32)) & 1u)) s[c / 64][c % 64] = __float_as_uint(-INFINITY);
        }
        float x0 = -INFINITY, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
#pragma unroll
        for (int c = 0; c < kBlock; c += 8) {
          x0 = fmax3(x0, __uint_as_float(s[c / 64][c % 64 + 0]), __uint_as_float(s[c / 64][c % 64 + 1]));
          x1 = fmax3(x1, __uint_as_float(s[c / 64][c % 64 + 2]), __uint_as_float(s[c / 64][c % 64 + 3]));
          x2 = fmax3(x2, __uint_as_float(s[c / 64][c % 64 + 4]), __uint_as_float(s[c / 64][c % 64 + 5]));
          x3 = fmax3(x3, __uint_as_float(s[c / 64][c % 64 + 6]), __uint_as_float(s[c / 64][c % 64 + 7]));
        }
        const float top = fmax3(x0, x1, fmaxf(x2, x3)) * p.item_scale;
        const bool need = top > m + kRescale;
        float alpha = 1.0f;
        if (need) {
          alpha = m == -INFINITY ? 0.0f : fast_exp2(m - top);
          l *= alpha;
          m = top;
        }
        if (x > 0 && __any_sync(0xffffffffu, need)) {
          // O's last update was issued before these scores, whose commit covers it
          for (int cb = 0; cb < D / 32; ++cb) {
            uint32_t o[32];
            tmem_ld32(o_tm + 32 * cb, o);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
            tmem_st32(o_tm + 32 * cb, o);
          }
        }
        const float sub = m == -INFINITY ? 0.0f : m;
        const uint64_t sc2 = f2(p.item_scale, p.item_scale), nm2 = f2(-sub, -sub);
        uint64_t l0 = f2(0.0f, 0.0f), l1 = l0;
        // P's two halves are handed over one by one: the first one's product runs during
        // the second one's exponentials
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            float y0, y1;
            f2_split(ffma2(f2(__uint_as_float(s[part][c]), __uint_as_float(s[part][c + 1])), sc2, nm2), y0, y1);
            y0 = fast_exp2(y0);
            y1 = fast_exp2(y1);
            if (c & 2) l1 = fadd2(l1, f2(y0, y1));
            else l0 = fadd2(l0, f2(y0, y1));
            pk[c / 2] = pack_bf16x2(y0, y1);
          }
          tmem_st32(s_tm + 32 * part, pk);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (!rehearse && lane == 0) mbar_arrive(&bars.p_full[t][part]);
        }
        float a0, a1;
        f2_split(fadd2(l0, l1), a0, a1);
        l += a0 + a1;
        if (!rehearse) ++steps;
      }
      if (!ok) {
        if (lane == 0) give_up(p, 71);
        break;
      }
      if (rehearse) continue;
      ok = __all_sync(0xffffffffu, mbar_wait(&bars.o_full, k & 1, p.wait_limit));
      if (!ok) {
        if (lane == 0) give_up(p, 72);
        break;
      }
      tc_fence_after();
      // Two block streams hold the same rows: each warpgroup adds up half of the columns
      // of both, with m and l exchanged through TMEM (a row is the same lane in both).
      // The next item's products wait for both warpgroups' q_ready.
      float mine = 1.0f, theirs = 0.0f;                 // weights of the two streams' O
      if (!two) {
        tmem_st2(s_tm, __float_as_uint(m), __float_as_uint(l));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.merge[t]);
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.merge[1 - t], merges & 1, p.wait_limit));
        if (!ok) {
          if (lane == 0) give_up(p, 73);
          break;
        }
        ++merges;
        tc_fence_after();
        uint32_t u0, u1;
        tmem_ld2(tmem + lane_base + kColS + 128 * (1 - t), u0, u1);
        tmem_ld_wait();
        const float m2 = __uint_as_float(u0), l2 = __uint_as_float(u1), M = fmaxf(m, m2);
        const float base = M == -INFINITY ? 0.0f : M;
        mine = fast_exp2(m - base);
        theirs = fast_exp2(m2 - base);
        l = mine * l + theirs * l2;
        m = M;
      }
      // infinite or NaN values of tree slots were taken out of V: the rows that see them get
      // them from the cache
      const bool odd = it.own && (bars.odd[k & 3][0] | bars.odd[k & 3][1]) != 0;
      // the part: O as [column quad][row] so that a warp stores 512 contiguous bytes
      float* part = p.parts + (int64_t)index * S::kPartFloats + (two ? t * (S::kPartFloats / 2) : 0);
      const int cb0 = two ? 0 : t * (D / 64), cb1 = two ? D / 32 : cb0 + D / 64;
#pragma unroll 1
      for (int cb = cb0; cb < cb1; ++cb) {
        uint32_t o[32];
        tmem_ld32(o_tm + 32 * cb, o);
        if (!two) {
          uint32_t o2[32];
          tmem_ld32(tmem + lane_base + kColO + D * (1 - t) + 32 * cb, o2);
          tmem_ld_wait();
          // a stream that has had no block (weight 0) has no O
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float x = mine != 0.0f ? mine * __uint_as_float(o[c]) : 0.0f;
            o[c] = __float_as_uint(theirs != 0.0f ? fmaf(theirs, __uint_as_float(o2[c]), x) : x);
          }
        }
        tmem_ld_wait();
        if (odd && valid) {
          for (int col = max(it.ja * kBlock, it.prefix); col < min(it.jb * kBlock, it.tokens); ++col) {
            if (!(seen_columns(a, it.tok0 + node, node, col & ~63, it.prefix, it.tokens) >> (col & 63) & 1ull)) continue;
            const int pg = p.page_of(col), page = a.page_indices[it.table + pg];
            if (page < 0 || page >= a.max_pages) continue;
            const uint16_t* v = (const uint16_t*)a.kv +
                                (((int64_t)page * 2 + 1) * a.page_len + (col - pg * a.page_len)) * a.Hkv * D +
                                (int64_t)it.h * D + 32 * cb;
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const float y = bf16_bits_to_float(v[c]);
              if (!(fabsf(y) < INFINITY)) o[c] = __float_as_uint(__uint_as_float(o[c]) + y);
            }
          }
        }
        if (valid) {
#pragma unroll
          for (int qd = 0; qd < 8; ++qd)
            *(float4*)(part + ((cb * 8 + qd) * 128 + r_local) * 4) =
                make_float4(__uint_as_float(o[4 * qd]), __uint_as_float(o[4 * qd + 1]),
                            __uint_as_float(o[4 * qd + 2]), __uint_as_float(o[4 * qd + 3]));
        }
      }
      tc_fence_before();
      if (valid && (two || t == 0)) {
        part[128 * D + r_local] = m;
        part[128 * D + 128 + r_local] = l;
      }
    }
  } else {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kHelperRegs));
  if (warp == 0) {
    // ------------------------------------------------------------ items and TMA producer
    // Item k + 1 is claimed when item k's last copies have been issued, a ring's length
    // before it ends (any earlier, a CTA holds a second item while others have none).
    // Lane r brings the r-th copy of a block.  The page of load x + 4 is fetched while load x is issued (unrolled by four,
    // so that no register that a fetch is still filling is moved).
    pdl_wait();
    const int total = __ldcg(&p.head->total);
    const int copies = kBlock / p.copy_tokens;
    bool ok = true;
    int pushed = 0, mine = blockIdx.x;                  // copies into the ring so far; this item's number
    for (int k = 0; ok; ++k) {
      const bool more = mine < total;
      const Item it = p.items[min(mine, p.max_items - 1)];   // (read beside the total, not after it)
      // the slot's last item, k - 2, has been copied by everyone
      ok = k < 2 || __all_sync(0xffffffffu, mbar_wait(&bars.item_free[k & 1], ((k >> 1) + 1) & 1, p.wait_limit));
      if (!ok) break;
      if (lane == 0) {
        bars.index[k & 1] = more ? mine : -1;
        if (more) bars.items[k & 1] = it;
        mbar_arrive(&bars.item_full[k & 1]);
      }
      __syncwarp();
      if (!more) break;
      const bool two = it.rows > 128;
      const int n = it.jb - it.ja;
      const int32_t* table = a.page_indices + it.table;
      // the x-th load: K or V, and this lane's token of it
      auto what = [&](int x, bool& is_v, int& tok) {
        int j;
        if (two) {                                      // K0 V0 K1 V1 ..
          is_v = x & 1;
          j = x >> 1;
        } else if (x < min(2, n)) {                     // K0 K1 V0 K2 V1 .. , the last two V
          is_v = false;
          j = x;
        } else {
          is_v = x == 2 * n - 1 || !(x & 1);
          j = x == 2 * n - 1 ? n - 1 : is_v ? (x - 2) / 2 : (x + 1) / 2;
        }
        tok = (it.ja + j) * kBlock + (lane & (copies - 1)) * p.copy_tokens;
      };
      auto fetch = [&](int x) -> int {
        bool is_v;
        int tok;
        what(x, is_v, tok);
        return x < 2 * n && tok < it.tokens ? __ldg(table + p.page_of(tok)) : -1;
      };
      auto push = [&](int x, int page) {
        bool is_v;
        int tok;
        what(x, is_v, tok);
        const int s = pushed % S::kSlots;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.empty[s], ((pushed / S::kSlots) + 1) & 1, p.wait_limit));
        if (!ok) return;
        if (page < 0 || page >= a.max_pages) page = a.max_pages;    // past the pool: zero fill
        if (lane == 0) mbar_arrive_expect_tx(&bars.full[s], S::kSlotBytes);
        __syncwarp();
        if (lane < copies)
          tma_load_5d(smem + S::kOffRing + s * S::kSlotBytes + lane * (p.copy_tokens / 8) * S::kGroupBytes, &kv_map,
                      &bars.full[s], 0, 0, it.h * S::kHalves, (tok - p.page_of(tok) * a.page_len) / 8,
                      2 * page + (is_v ? 1 : 0));
        __syncwarp();
        ++pushed;
      };
      int p0 = fetch(0), p1 = fetch(1), p2 = fetch(2), p3 = fetch(3);
      for (int x = 0; ok && x < 2 * n; x += 4) {
        push(x, p0);
        p0 = fetch(x + 4);
        if (!ok || x + 1 >= 2 * n) break;
        push(x + 1, p1);
        p1 = fetch(x + 5);
        if (!ok || x + 2 >= 2 * n) break;
        push(x + 2, p2);
        p2 = fetch(x + 6);
        if (!ok || x + 3 >= 2 * n) break;
        push(x + 3, p3);
        p3 = fetch(x + 7);
      }
      if (lane == 0) mine = atomicAdd(&p.head->next, 1);
      mine = __shfl_sync(0xffffffffu, mine, 0);
    }
    if (!ok && lane == 0) give_up(p, 51);
    // the copies in flight must land before the CTA can exit
    for (int x = max(0, pushed - S::kSlots); x < pushed; ++x)
      mbar_wait(&bars.full[x % S::kSlots], (x / S::kSlots) & 1);
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer, one thread
    if (elect_one()) {
      const uint32_t id_qk = idesc_bf16_f32(128, kBlock, 0, 0);
      const uint32_t id_pv = idesc_bf16_f32(128, D, 0, 1);
      // eight-token groups kGroupBytes apart, a group's halves 1 KB
      const uint64_t q0 = smem_desc(smem_u32(smem + S::kOffQ), 16, 1024, kSwizzle128B);
      const uint64_t k0 = smem_desc(smem_u32(smem + S::kOffRing), 16, S::kGroupBytes, kSwizzle128B);
      const uint64_t v0 = smem_desc(smem_u32(smem + S::kOffRing), 1024, S::kGroupBytes, kSwizzle128B);
      bool ok = true, issued = false;
      int base = 0, steps0 = 0, steps1 = 0;             // ring positions before this item; blocks done
      int arrived = 0, passed = 0;                      // masked value blocks announced; used up
      auto wait = [&](uint64_t* bar, int parity, int code) {
        ok = ok && mbar_wait(bar, parity & 1, p.wait_limit);
        if (!ok) give_up(p, code);
        return ok;
      };
      Item it;
      for (int k = 0; ok && next_item(k, it); ++k) {
        mbar_arrive(&bars.item_free[k & 1]);
        const bool two = it.rows > 128;
        const int n = it.jb - it.ja;
        const int count0 = two ? n : (n + 1) / 2, count1 = two ? n : n / 2;
        if (!wait(&bars.q_ready, k, 61)) break;
        // step 2 x + t: O += P V of stream t's block x - 1, then S = Q K^T of its block x
        for (int st = 0; ok && st < 2 * (count0 + 1); ++st) {
          const int t = st & 1, x = st >> 1, count = t ? count1 : count0;
          if (x > count) continue;
          const int kpos = base + ring_k(two, two ? x : 2 * x + t), kslot = kpos % S::kSlots;
          // K of the next scores first: it is there long before P is
          if (x < count && !wait(&bars.full[kslot], kpos / S::kSlots, 65)) break;
          if (x > 0) {
            const int blk = two ? x - 1 : 2 * (x - 1) + t;
            const int pos = base + ring_v(two, blk, n), slot = pos % S::kSlots;
            if (!wait(&bars.full[slot], pos / S::kSlots, 63)) break;
            if (masked_block(it, blk)) {
              // warps 2 and 3 have gone over the block's values
              const long long since = clock64();
              while (bars.cleaned[0] <= passed || bars.cleaned[1] <= passed)
                if (clock64() - since > p.wait_limit) {
                  ok = false;
                  break;
                }
              if (!ok) {
                give_up(p, 66);
                break;
              }
              if (!two || t == 1) ++passed;
            }
            const uint64_t vd = v0 + (uint64_t)((slot * S::kSlotBytes) >> 4);
            const int ph = (t ? steps1++ : steps0++) & 1;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              ok = mbar_wait_spin(&bars.p_full[t][part], ph, p.wait_limit);
              if (!ok) {
                give_up(p, 64);
                break;
              }
              tc_fence_after();
#pragma unroll
              for (int j = part * kRuns / 2; j < (part + 1) * kRuns / 2; ++j)
                mma_bf16_ts(tmem + kColO + D * t, tmem + kColS + 128 * t + 8 * j,
                            vd + (uint64_t)((j * S::kRunBytes) >> 4), id_pv, (x > 1 || j > 0) ? 1u : 0u);
            }
            if (!ok) break;
            if (!two || t == 1) mma_commit(&bars.empty[slot]);
          }
          if (x < count) {
            tc_fence_after();
            const uint64_t qd = q0 + (uint64_t)((two ? t * S::kSlotBytes : 0u) >> 4);
            const uint64_t kd = k0 + (uint64_t)((kslot * S::kSlotBytes) >> 4);
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
              mma_bf16_ss(tmem + kColS + 128 * t, qd + (uint64_t)(((j / 4) * S::kQHalfBytes + (j % 4) * 32) >> 4),
                          kd + (uint64_t)(((j / 4) * 1024 + (j % 4) * 32) >> 4), id_qk, j > 0);
            mma_commit(&bars.s_full[t]);
            if (!two || t == 1) mma_commit(&bars.empty[kslot]);
            issued = true;
            const int blk = two ? x : 2 * x + t;
            if (masked_block(it, blk) && (!two || t == 0)) {
              // its values come right behind the keys: warps 2 and 3 may start on them
              const int pos = base + ring_v(two, blk, n);
              if (!wait(&bars.full[pos % S::kSlots], pos / S::kSlots, 67)) break;
              __threadfence_block();
              bars.arrived = ++arrived;
            }
          }
        }
        if (ok) mma_commit(&bars.o_full);
        base += 2 * n;
      }
      if (issued) {
        mma_commit(&bars.drain);
        mbar_wait(&bars.drain, 0);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ values of masked slots
    // A masked probability is 0, and 0 * v is 0 only for finite v.  Warps 2 and 3 each go
    // over half the tokens of an own item's masked value blocks while the scores' softmax
    // runs: slots from the length on (the rest of a page) are zeroed, and so are infinite
    // or NaN values of tree slots, which is noted for the rows that do see them.
    const int half = warp - 2;
    bool ok = true;
    int base = 0, done = 0;                             // ring positions before this item; masked blocks so far
    Item it;
    for (int k = 0; ok; ++k) {
      if (!__all_sync(0xffffffffu, next_item(k, it))) break;
      if (lane == 0) {
        bars.odd[k & 3][half] = 0;
        mbar_arrive(&bars.item_free[k & 1]);
      }
      const bool two = it.rows > 128;
      const int n = it.jb - it.ja;
      for (int j = it.own ? max(0, max(it.prefix, 0) / kBlock - it.ja) : n; ok && j < n; ++j) {
        const int c0 = (it.ja + j) * kBlock, pos = base + ring_v(two, j, n), slot = pos % S::kSlots;
        // the MMA thread has seen the block arrive; it is not overwritten before this
        // warp has passed it, so the barrier's phase is this block's
        const long long since = clock64();
        while (bars.arrived <= done && ok) ok = clock64() - since <= p.wait_limit;
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars.full[slot], (pos / S::kSlots) & 1, p.wait_limit));
        if (!ok) break;
        const uint32_t vb = smem_u32(smem + S::kOffRing + slot * S::kSlotBytes);
        auto at = [&](int x) -> uint32_t {                // 16-byte piece x of the block's values, token by token
          const int tok = x / (D / 8), ch = x % (D / 8);
          return vb + (tok >> 3) * S::kGroupBytes + (ch >> 3) * 1024 + (tok & 7) * 128 + (((ch & 7) ^ (tok & 7)) << 4);
        };
        const int lo = max(half * 64, it.prefix - c0);  // tokens before it are the prefix
        const int end = min((half + 1) * 64, max(lo, it.tokens - c0)), stop = end * (D / 8);
        for (int x = lo * (D / 8) + lane; x < stop; x += 32 * 8) {
          uint4 v[8];                                   // eight pieces in flight
#pragma unroll
          for (int u = 0; u < 8; ++u) v[u] = x + 32 * u < stop ? ld_shared_v4(at(x + 32 * u)) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            if (odd2(v[u].x) || odd2(v[u].y) || odd2(v[u].z) || odd2(v[u].w)) {
              auto fix = [](uint32_t w) {
                if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
                if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
                return w;
              };
              st_shared_v4(at(x + 32 * u), fix(v[u].x), fix(v[u].y), fix(v[u].z), fix(v[u].w));
              bars.odd[k & 3][half] = 1;
            }
          }
        }
        for (int x = max(end, half * 64) * (D / 8) + lane; x < (half + 1) * 64 * (D / 8); x += 32)
          if (c0 + x / (D / 8) >= it.tokens) st_shared_v4(at(x), 0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
        __threadfence_block();
        __syncwarp();
        ++done;
        if (lane == 0) bars.cleaned[half] = done;
      }
      base += 2 * n;
    }
    if (!ok && lane == 0) give_up(p, 91);
  }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ----------------------------------------------------------------------- joining
__device__ __forceinline__ Entry load_entry(const Entry* e) {
  const int4 x = __ldcg((const int4*)e), y = __ldcg((const int4*)e + 1);
  return Entry{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
}

// A CTA joins 16 rows of a request and KV head: the parts of its group's shared columns,
// and those of its own.  A thread has a row and a column quad -- four rows and eight
// quads per warp, so that both the parts ([quad][row]) and the output are touched in
// 64-byte pieces -- and, with few rows, every slices-th of the parts.  Bound by the
// latency of reading what other SMs have just written: the first O values are asked for
// together with the parts' m and l, which become weights e^(m - M) meanwhile.  256 rows of
// 8 KV heads with 17 parts each (18 MB): 5-7 us.
constexpr int kJoinRows = 16;
constexpr int kJoinThreads = 256;
constexpr int kJoinAhead = 6;             // O values in flight per thread
constexpr int kMaxParts = 2 * kMaxSplits;
static_assert(kMaxOwnSplits <= kMaxSplits, "");

template <int D>
__global__ void __launch_bounds__(kJoinThreads, 4) join_parts_kernel(const PrefixParams p, int row_tiles) {
  const SharedAttnParams& a = p.a;
  constexpr int kPart = Shape<D>::kPartFloats, kHalf = kPart / 2;
  __shared__ float w[kMaxParts][kJoinRows], lw[kMaxParts][kJoinRows];
  __shared__ float inv[kJoinRows];
  __shared__ float4 sum[kJoinThreads];
  pdl_trigger();
  const int b = blockIdx.x / row_tiles, row0 = (blockIdx.x - b * row_tiles) * kJoinRows, h = blockIdx.y;
  const int tok0 = a.qo_indptr[b], total_rows = (a.qo_indptr[b + 1] - tok0) * a.g, gi = group_of(a, b);
  pdl_wait();                                           // (the lengths are no kernel's of this call)
  if (row0 >= total_rows) return;
  const int n = min(kJoinRows, total_rows - row0);
  // A stored part is [quad][128 rows] with m and l behind; own_attn_kernel's are [quad] with
  // (m, l) apart.
  const Entry group = p.entries[gi];
  const int shared = group.splits, parts = shared + p.own_splits;
  auto part_of = [&](const Entry& e, int R, int& in) -> const float* {   // the first part's half with row R, its place
    const int at = (tok0 - e.tok0) * a.g + R, tile = at / kTileRows;
    in = at & 127;
    return p.parts + ((int64_t)e.first + ((int64_t)h * tiles_of(e.rows) + tile) * e.splits) * kPart +
           ((at >> 7) & 1) * kHalf;
  };
  auto row_of = [&](int R) -> int64_t {
    const int tk = p.div_g.div(R);
    return (int64_t)(tok0 + tk) * a.Hq + h * a.g + R - tk * a.g;
  };
  const int units = (n + 3) / 4 * D, slices = max(1, kJoinThreads / units);
  // this thread's place in round `idx`: row, quad, first parts
  int r = 0, quad = 0;
  const float *s0 = nullptr, *s1 = nullptr;
  auto place = [&](int unit) {
    const int lo = unit & 31, hi = unit >> 5;
    r = (hi / (D / 32)) * 4 + (lo & 3);
    quad = (hi % (D / 32)) * 8 + (lo >> 2);
    const int R = row0 + min(r, n - 1);
    int in;
    s0 = part_of(group, R, in);
    s0 += quad * 512 + in * 4;
    s1 = p.own_o + row_of(R) * p.own_splits * D + quad * 4;
  };
  float4 v[kJoinAhead];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      const int k = k0 + u * slices;
      if (k < parts) v[u] = __ldcg((const float4*)(k < shared ? s0 + (int64_t)k * kPart : s1 + (int64_t)(k - shared) * D));
    }
  };
  int idx = threadIdx.x;
  const bool busy = idx < units * slices;
  if (busy) {
    place(idx % units);
    fetch(idx / units);
  }
#pragma unroll 2
  for (int e = threadIdx.x; e < parts * kJoinRows; e += kJoinThreads) {
    const int rr = e % kJoinRows, k = e / kJoinRows, R = row0 + rr;
    float m = -INFINITY, l = 0.0f;
    if (rr < n) {
      if (k >= shared) {
        const float2 x = __ldcg(p.own_ml + row_of(R) * p.own_splits + (k - shared));
        m = x.x;
        l = x.y;
      } else {
        int in;
        const float* s = part_of(group, R, in) + (int64_t)k * kPart;
        m = __ldcg(s + 128 * D + in);
        l = __ldcg(s + 128 * D + 128 + in);
      }
    }
    w[k][rr] = m;
    lw[k][rr] = l;
  }
  __syncthreads();
  {
    // sixteen threads per row
    const int rr = threadIdx.x / 16, j = threadIdx.x % 16;
    float M = -INFINITY, L = 0.0f;
    for (int k = j; k < parts; k += 16) M = fmaxf(M, w[k][rr]);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    const float base = M == -INFINITY ? 0.0f : M;
    for (int k = j; k < parts; k += 16) {
      const float x = fast_exp2(w[k][rr] - base);
      L = fmaf(x, lw[k][rr], L);
      w[k][rr] = x;
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
    if (j == 0) inv[rr] = L > 0.0f ? 1.0f / L : L == L ? 0.0f : L;   // nothing seen: 0
  }
  __syncthreads();
  for (; idx < units * slices; idx += kJoinThreads) {
    const int unit = idx % units, slice = idx / units;
    if (idx != (int)threadIdx.x) {
      place(unit);
      fetch(slice);
    }
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k0 = slice; k0 < parts; k0 += kJoinAhead * slices) {
      if (k0 != slice) fetch(k0);
#pragma unroll
      for (int u = 0; u < kJoinAhead; ++u) {
        const int k = k0 + u * slices;
        const float x = k < parts ? w[k][r] : 0.0f;
        if (x != 0.0f) {                                // a part of no columns has no O
          o.x = fmaf(x, v[u].x, o.x);
          o.y = fmaf(x, v[u].y, o.y);
          o.z = fmaf(x, v[u].z, o.z);
          o.w = fmaf(x, v[u].w, o.w);
        }
      }
    }
    if (slices > 1) {                                   // (then units * slices is the CTA's threads: one round)
      sum[idx] = o;
      __syncthreads();
      if (slice > 0) return;
      for (int i = 1; i < slices; ++i) {
        const float4 y = sum[unit + i * units];
        o.x += y.x;
        o.y += y.y;
        o.z += y.z;
        o.w += y.w;
      }
    }
    if (r >= n) continue;
    const float f = inv[r];
    *(uint2*)((uint16_t*)a.out + row_of(row0 + r) * D + quad * 4) =
        make_uint2(pack_bf16x2(o.x * f, o.y * f), pack_bf16x2(o.z * f, o.w * f));
  }
}

// The same where own columns are work items: many rows and few parts, so a warp takes four
// rows, and a lane the quads q, q + 8, .. of one; a part's m, l and O are all asked for at
// once, and the sums are rescaled as the maximum grows.  3500 rows of 8 KV heads with two
// parts each (29 MB and 7 MB of output): 10 us, 16 from a cold cache; through the kernel
// above, two barriers between its loads, 18.
constexpr int kTilesThreads = 128;

template <int D>
__global__ void __launch_bounds__(kTilesThreads, 8) join_tiles_kernel(const PrefixParams p, int row_tiles) {
  constexpr int kPart = Shape<D>::kPartFloats, kHalf = kPart / 2, kQuads = D / 32;
  const SharedAttnParams& a = p.a;
  const int lane = threadIdx.x & 31;
  pdl_trigger();
  const int b = blockIdx.x / row_tiles, h = blockIdx.y;
  const int row0 = (blockIdx.x - b * row_tiles) * kJoinRows + threadIdx.x / 32 * 4;
  const int tok0 = a.qo_indptr[b], rows = (a.qo_indptr[b + 1] - tok0) * a.g, group = group_of(a, b);
  pdl_wait();                                           // (the lengths are no kernel's of this call)
  if (row0 >= rows) return;
  const Entry shared = load_entry(p.entries + group), own = load_entry(p.entries + a.groups + b);
  const int r = min(row0 + (lane & 3), rows - 1), R = r + (tok0 - shared.tok0) * a.g, from = p.tail_from(rows);
  const bool tail = row0 >= from;                       // (whole warps: a tile's rows are a multiple of four)
  const int parts = shared.splits + (tail ? p.own_splits : own.splits);
  const int64_t tail_part = (((int64_t)b * a.Hkv + h) * kFewRows + r - from) * p.own_splits;
  auto part_of = [&](const Entry& e, int at) -> const float* {
    return p.parts + ((int64_t)e.first + (int64_t)(h * tiles_of(e.rows) + at / kTileRows) * e.splits) * kPart +
           ((at >> 7) & 1) * kHalf + (at & 127);
  };
  const float *s0 = part_of(shared, R), *s1 = part_of(own, r);
  float M = -INFINITY, L = 0.0f;
  float4 acc[kQuads];
#pragma unroll
  for (int j = 0; j < kQuads; ++j) acc[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 2
  for (int k = 0; k < parts; ++k) {
    float m, l;
    float4 v[kQuads];
    if (tail && k >= shared.splits) {
      const int64_t part = tail_part + (k - shared.splits);
      const float2 x = __ldcg(p.own_ml + part);
      m = x.x;
      l = x.y;
#pragma unroll
      for (int j = 0; j < kQuads; ++j) v[j] = __ldcg((const float4*)(p.own_o + part * D) + 8 * j + (lane >> 2));
    } else {
      const float* s = k < shared.splits ? s0 + (int64_t)k * kPart : s1 + (int64_t)(k - shared.splits) * kPart;
      const int in = (k < shared.splits ? R : r) & 127;
      m = __ldcg(s + 128 * D);
      l = __ldcg(s + 128 * D + 128);
#pragma unroll
      for (int j = 0; j < kQuads; ++j) v[j] = __ldcg((const float4*)(s - in + (8 * j + (lane >> 2)) * 512 + in * 4));
    }
    const float top = fmaxf(M, m), base = top == -INFINITY ? 0.0f : top;
    const float f = fast_exp2(M - base), w = fast_exp2(m - base);
    L = f * L + w * l;
    M = top;
    // a part of no columns has no O
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
      acc[j].x = (f != 0.0f ? f * acc[j].x : 0.0f) + (w != 0.0f ? w * v[j].x : 0.0f);
      acc[j].y = (f != 0.0f ? f * acc[j].y : 0.0f) + (w != 0.0f ? w * v[j].y : 0.0f);
      acc[j].z = (f != 0.0f ? f * acc[j].z : 0.0f) + (w != 0.0f ? w * v[j].z : 0.0f);
      acc[j].w = (f != 0.0f ? f * acc[j].w : 0.0f) + (w != 0.0f ? w * v[j].w : 0.0f);
    }
  }
  if (row0 + (lane & 3) >= rows) return;
  const float c = L > 0.0f ? 1.0f / L : L == L ? 0.0f : L;        // nothing seen: 0
  const int tk = p.div_g.div(r);
  uint16_t* out = (uint16_t*)a.out + ((int64_t)(tok0 + tk) * a.Hq + h * a.g + r - tk * a.g) * D + (lane >> 2) * 4;
#pragma unroll
  for (int j = 0; j < kQuads; ++j)
    *(uint2*)(out + 32 * j) = make_uint2(pack_bf16x2(acc[j].x * c, acc[j].y * c), pack_bf16x2(acc[j].z * c, acc[j].w * c));
}

struct PrefixPlan {
  int few, direct, narrow, tail_rows, own_rows, own_splits, max_items, ctas;
  size_t head, entries, items, parts, own_ml, own_o, bytes;
};

int sm_count() {
  static std::atomic<int> counts[64];                   // per device
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  n = counts[dev].load();
  if (n) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
  counts[dev].store(n);
  return n;
}

PrefixPlan plan_prefix(int batch, int groups, int total_q, int max_qo_len, int max_kv_len, int max_own_len, int Hq,
                       int Hkv, int D) {
  PrefixPlan f;
  const int g = Hq / Hkv;
  const int64_t rows = (int64_t)max_qo_len * g;
  f.few = rows <= kFewRows;
  // A tree of a few rows more than whole tiles has a tile for them, which costs a CTA almost
  // as much as a full one: own_attn_kernel takes them beside it instead (and those of the
  // other requests).  16 requests of 260 rows per KV head after 4096 shared tokens: 102 us with
  // it, 114 without; of 516 rows 190 and 195; 4 of 260 rows 52 and 60.  Half tiles do
  // not gain by it (132 rows: 62 and 61, with 1500 own tokens 113 and 104).
  f.tail_rows = !f.few && rows % kTileRows && rows % kTileRows <= kFewRows ? kFewRows : 0;
  f.own_rows = rows <= 8 ? 8 : 16;
  f.ctas = sm_count();
  // One launch that reads each request's columns takes about 3 us + 5 ns a token for each
  // round of (request, KV head) pairs over the SMs.  It and the other way, in us: 512
  // tokens 6.6 and 16.1 with 48 pairs of head_dim 64, 7.9 and 18.6 with 128 of 128; 1900
  // tokens 12.1 and 17.6, 14.2 and 21.8; 1100 tokens, 240 pairs of 128 19.3 and 21.5.
  f.direct = f.few && ((batch * (int64_t)Hkv + f.ctas - 1) / f.ctas) * (600 + (int64_t)max_kv_len) <= kDirectCost;
  if (f.direct) {
    f.own_splits = 1;
    f.max_items = 0;
    f.head = f.entries = f.items = f.parts = f.own_ml = f.own_o = 0;
    f.bytes = 0;
    return f;
  }
  // own columns: slices for about six CTAs of two warps per SM, each warp with two runs at least
  const int own = max_own_len > 0 ? max_own_len : max_kv_len;
  // Decoding with more own columns than shared ones: prefix_attn_kernel gives a slot of its ring
  // to a second own_attn_kernel CTA beside it.  64 requests of 8192 shared and 300 own tokens
  // 41.7 us with it, 46.1 without; 32 of 65536 and 500 85.9 and 77.7.
  f.narrow = f.few && max_own_len > 0 && (int64_t)batch * max_own_len >= (int64_t)groups * (max_kv_len - max_own_len);
  f.own_splits = 1;
  if (f.few || f.tail_rows)
    f.own_splits = (int)std::max<int64_t>(1, std::min<int64_t>({6ll * f.ctas / std::max<int64_t>((int64_t)batch * Hkv, 1),
                                                                ((int64_t)own + 4 * kRun - 1) / (4 * kRun), kMaxOwnSplits}));
  int64_t units = ((int64_t)total_q * g + kTileRows - 1) / kTileRows + groups;
  if (!f.few) units += ((int64_t)total_q * g + kTileRows - 1) / kTileRows + batch;
  f.max_items = (int)std::min<int64_t>(units * Hkv + 2 * f.ctas, 1 << 28);
  const int part = D == 128 ? Shape<128>::kPartFloats : Shape<64>::kPartFloats;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at = align_up(at + n, 256);
    return o;
  };
  f.head = take(sizeof(PlanHead));
  f.entries = take(sizeof(Entry) * (groups + (f.few ? 0 : batch)));
  f.items = take(sizeof(Item) * f.max_items);
  f.parts = take((size_t)f.max_items * part * sizeof(float));
  const size_t own_parts = (f.few ? (size_t)total_q * Hq : f.tail_rows ? (size_t)batch * Hkv * kFewRows : 0) * f.own_splits;
  f.own_ml = take(own_parts * sizeof(float2));
  f.own_o = take(own_parts * D * sizeof(float));
  f.bytes = at;
  return f;
}

template <int D>
int encode_kv(CUtensorMap* map, const SharedAttnParams& a, int copy_tokens) {
  // (dim of a half, token of a group, head and half, group, 2 page + K/V)
  const cuuint64_t tok = (cuuint64_t)a.Hkv * D * 2;
  const cuuint64_t dims[5] = {64, 8, (cuuint64_t)a.Hkv * (D / 64), (cuuint64_t)a.page_len / 8, (cuuint64_t)a.max_pages * 2};
  const cuuint64_t strides[4] = {tok, 128, 8 * tok, a.page_len * tok};
  const cuuint32_t box[5] = {64, 8, D / 64, (cuuint32_t)copy_tokens / 8, 1};
  return encode_tiled_bf16_sw128(map, 5, a.kv, dims, strides, box);
}

template <int D, int NR, int NW, bool kDirect>
int launch_own(const PrefixParams& p, const CUtensorMap& map, cudaStream_t stream) {
  constexpr size_t smem = own_smem<D, NR, NW>();
  auto kernel = own_attn_kernel<D, NR, NW, kDirect>;
  if (int rc = ensure_smem_attr((const void*)kernel, smem, true)) return rc;
  PTS_CUDA_TRY(launch_pdl(kernel, dim3(p.a.batch, p.a.Hkv, p.own_splits), dim3(32 * NW), smem, stream, p, map));
  return launch_status("own_attn_kernel");
}

template <int D, int SLOTS>
int launch_items(const PrefixParams& p, const PrefixPlan& f, const CUtensorMap& map, cudaStream_t stream) {
  auto kernel = prefix_attn_kernel<D, SLOTS>;
  constexpr size_t smem = Shape<D, SLOTS>::kSmem;
  if (int rc = ensure_smem_attr((const void*)kernel, smem, true)) return rc;
  // setmaxnreg.inc would wait for good for registers that the launch does not have
  static std::atomic<int> regs{0};
  if (!regs.load()) {
    cudaFuncAttributes attr;
    PTS_CUDA_TRY(cudaFuncGetAttributes(&attr, (const void*)kernel));
    regs.store(attr.numRegs);
  }
  if (regs.load() < kLaunchRegs)
    return set_error(PTS_ERR_CUDA, "prefix_attn_kernel was built with %d registers (%d needed)", regs.load(), kLaunchRegs);
  PTS_CUDA_TRY(launch_pdl(kernel, dim3(f.ctas), dim3(kThreads), smem, stream, p, map));
  return launch_status("prefix_attn_kernel");
}

template <int D>
int launch_prefix(const PrefixParams& p, const PrefixPlan& f, int max_qo_len, cudaStream_t stream) {
  CUtensorMap run_map, block_map;
  if (f.few || f.tail_rows)
    if (int rc = encode_kv<D>(&run_map, p.a, kRun)) return rc;
  if (f.direct)
    return f.own_rows == 8 ? launch_own<D, 1, kDirectWarps, true>(p, run_map, stream)
                           : launch_own<D, 2, kDirectWarps, true>(p, run_map, stream);
  if (int rc = encode_kv<D>(&block_map, p.a, p.copy_tokens)) return rc;
  // (the small kernels ask for the same shared-memory split, which an SM changes only when idle)
  if (int rc = ensure_smem_attr((const void*)plan_kernel, 1, true)) return rc;
  if (int rc = ensure_smem_attr(f.few ? (const void*)join_parts_kernel<D> : (const void*)join_tiles_kernel<D>, 1, true))
    return rc;
  PTS_CUDA_TRY(launch_pdl(plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p));
  if (int rc = launch_status("plan_kernel")) return rc;
  int rc = PTS_OK;
  if constexpr (D == 128)
    rc = f.narrow ? launch_items<D, 3>(p, f, block_map, stream) : launch_items<D, Shape<D>::kSlots>(p, f, block_map, stream);
  else
    rc = launch_items<D, Shape<D>::kSlots>(p, f, block_map, stream);
  if (rc) return rc;
  if (f.few || f.tail_rows)
    if (int rc = f.own_rows == 8 ? launch_own<D, 1, kOwnWarps, false>(p, run_map, stream)
                                 : launch_own<D, 2, kOwnWarps, false>(p, run_map, stream))
      return rc;
  const int row_tiles = (int)(((int64_t)max_qo_len * p.a.g + kJoinRows - 1) / kJoinRows);
  const dim3 grid(p.a.batch * row_tiles, p.a.Hkv);
  if (f.few) PTS_CUDA_TRY(launch_pdl(join_parts_kernel<D>, grid, dim3(kJoinThreads), 0, stream, p, row_tiles));
  else PTS_CUDA_TRY(launch_pdl(join_tiles_kernel<D>, grid, dim3(kTilesThreads), 0, stream, p, row_tiles));
  return launch_status("join_parts_kernel");
}

}  // namespace

bool prefix_attn_supports(int head_dim, int page_len, int elem_bytes) {
  return elem_bytes == 2 && (head_dim == 64 || head_dim == 128) && page_len % kRun == 0;
}

size_t prefix_attn_workspace(int batch, int groups, int total_q, int max_qo_len, int max_kv_len, int max_own_len,
                             int Hq, int Hkv, int D) {
  return plan_prefix(batch, groups, total_q, max_qo_len, max_kv_len, max_own_len, Hq, Hkv, D).bytes;
}

int prefix_attn_launch(const SharedAttnParams& a, int total_q, int max_qo_len, int max_kv_len, int max_own_len,
                       void* workspace, int32_t* error, cudaStream_t stream) {
  const PrefixPlan f = plan_prefix(a.batch, a.groups, total_q, max_qo_len, max_kv_len, max_own_len, a.Hq, a.Hkv, a.D);
  if ((int64_t)a.batch * ((int64_t)max_qo_len * a.g / kJoinRows + 1) > 2147483647ll)
    return set_error(PTS_ERR_CAPACITY, "grid too large");
  if ((int64_t)total_q * a.g * a.g > 0xffffffffll)
    return set_error(PTS_ERR_CAPACITY, "%d query rows are too many", total_q);
  char* ws = (char*)workspace;
  PrefixParams p{};
  p.a = a;
  p.div_g = FastDiv((uint32_t)a.g);
  p.copy_tokens = kRun;
  while (p.copy_tokens < kBlock && a.page_len % (2 * p.copy_tokens) == 0) p.copy_tokens *= 2;
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (a.page_len == 1 << s) p.page_shift = s;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.item_scale = fabsf(p.scale_log2) < FLT_MIN ? FLT_MIN : fabsf(p.scale_log2);
  p.flip = a.scale < 0.0f ? 0x80008000u : 0u;
  p.error = error;
  p.wait_limit = wait_limit_cycles();
  p.ctas = f.ctas;
  p.max_items = f.max_items;
  p.own_items = !f.few;
  p.tail_rows = f.tail_rows;
  p.head = (PlanHead*)(ws + f.head);
  p.entries = (Entry*)(ws + f.entries);
  p.items = (Item*)(ws + f.items);
  p.parts = (float*)(ws + f.parts);
  p.own_splits = f.own_splits;
  p.own_o = (float*)(ws + f.own_o);
  p.own_ml = (float2*)(ws + f.own_ml);
  return a.D == 128 ? launch_prefix<128>(p, f, max_qo_len, stream) : launch_prefix<64>(p, f, max_qo_len, stream);
}

}  // namespace pts
