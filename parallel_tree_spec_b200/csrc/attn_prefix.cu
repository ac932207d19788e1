// Tree attention for requests that share leading pages, bf16 with head_dim 64 or 128
// and pages of whole 16-token runs, on the tensor cores.  Two launches:
//
// prefix_attn_kernel: the shared columns, once for all rows of a group.  A group's
//   rows -- (token, query head of the KV head's group), its requests one after the
//   other -- are cut into tiles of 256; a work item is a row tile, a KV head and a
//   range of 128-token blocks.  Two streams of S = Q K^T, P = e^(S - m), O += P V run
//   in a CTA so that the tensor cores compute one's products while the other's
//   exponentials run: stream t holds rows 128 t .. 128 t + 127 of the tile, or, for
//   tiles of up to 128 rows (decoding a few dozen sequences), the same rows and every
//   second block.  tcgen05 with S and O in TMEM, P written back over S as the A operand
//   of the value product; K/V by TMA, a 16-token run at a time, into a ring; one
//   thread per row, so the softmax needs no shuffles.  Each item leaves one part per
//   row (fp32 O, m, l).
// own_attn_kernel: each request's own columns with its tree mask, then the join with
//   the shared parts.  A request has few rows (1 to 16 when decoding), far below the
//   tensor cores' 128-row tiles, and each of its K/V bytes is used by those rows only:
//   it is bound by HBM, so mma.sync m16n8k16 fed by cp.async is enough, and many small
//   CTAs per SM keep the loads in flight.  It starts while the first kernel runs
//   out (programmatic dependent launch) and waits for it before the join only.
//
// Scores are kept in units of log2: x = s * scale * log2(e), e^(s - m) = 2^(x - m').
#include <algorithm>

#include "attn_shared.cuh"
#include "sm100.cuh"

namespace pts {
namespace {

using namespace sm100;

constexpr int kBlock = 128;               // tokens per block
constexpr int kRun = 16;                  // tokens of one value product; pages are whole runs
constexpr int kRuns = kBlock / kRun;
constexpr int kTileRows = 256;
constexpr int kThreads = 384;             // warps 0 TMA, 1 MMA, 2-3 plan, 4-7 and 8-11 softmax
constexpr int kMaxSplits = 32;
constexpr int kPlanSmem = 40;             // groups whose plan fits in shared memory
constexpr float kRescale = 8.0f;          // O is rescaled when the row max grows by more than 2^8
constexpr uint32_t kColS = 0, kColO = 256;

// A block's K (or V) in shared memory: [8-token group][64-dim half][8 tokens][64 dims],
// 128-byte-swizzled rows.  One TMA copy brings a page's tokens (up to a block) with both
// halves, and the groups of a half lie evenly apart, as the matrix descriptors want.
template <int D>
struct Shape {
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kGroupBytes = kHalves * 1024;
  static constexpr uint32_t kRunBytes = 2 * kGroupBytes;
  static constexpr uint32_t kSlotBytes = kRuns * kRunBytes;     // K or V of a block; Q of a stream
  static constexpr uint32_t kQHalfBytes = 128 * 128;            // Q: [half][128 rows][64 dims]
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr uint32_t kOffQ = 0;
  static constexpr uint32_t kOffRing = 2 * kSlotBytes;
  static constexpr uint32_t kOffBars = kOffRing + kSlots * kSlotBytes;
  static constexpr uint32_t kSmem = kOffBars + 1280 + 1024;     // barriers, plan; alignment slack
  static constexpr int kPartFloats = 2 * 128 * (D + 2);         // one item's part: two streams' rows
};
static_assert(Shape<128>::kSmem <= 232448 && Shape<64>::kSmem <= 232448, "shared memory above 227 KB");

struct GroupPlan {
  int pages;      // shared pages
  int rows;       // query rows per KV head
  int tok0;       // the group's first token
  int table;      // where the page table of its first request with rows starts
  int first;      // first work item
  int splits;     // block ranges per (row tile, KV head)
};

// One work item.
struct Item {
  int h, tok0, table;       // KV head; first token of the group; its page table
  int rows, row0;           // rows of the tile: row0 .. of the group's rows per KV head
  int ja, jb, tokens;       // blocks; tokens of the shared columns
};

struct __align__(8) Bars {
  uint64_t q_ready;         // both warpgroups: done with the last item, this one's rows stored
  uint64_t full[8], empty[8];
  uint64_t s_full[2], p_full[2];
  uint64_t o_full, drain;
  uint32_t tmem;
  int chunk, total;         // blocks per range, work items
  Item first;               // this CTA's first item
  GroupPlan plan[kPlanSmem];
};
static_assert(sizeof(Bars) <= 1280, "barrier block");

struct PrefixParams {
  SharedAttnParams a;
  FastDiv div_g;
  int copy_tokens;          // tokens per TMA copy: the power of two in page_len, at most a block
  int page_shift;           // log2(page_len), or -1
  float scale_log2;
  int max_items;            // parts in the workspace
  float* parts;
  GroupPlan* plan;          // [groups], for the second kernel
  GroupPlan* cta_plan;      // [CTAs][groups] when the groups do not fit in shared memory
  int* error;
  long long wait_limit;
  // own columns
  int own_splits, request_tiles;
  float* own_o;             // [T * Hq][own_splits][D]
  float2* own_ml;           // [T * Hq][own_splits]

  __device__ __forceinline__ int page_of(int tok) const { return page_shift >= 0 ? tok >> page_shift : tok / a.page_len; }
};

__device__ __forceinline__ void give_up(const PrefixParams& p, int code) {
  if (p.error) atomicExch(p.error, code);
}

__device__ __forceinline__ int blocks_of(int pages, int page_len) { return (pages * page_len + kBlock - 1) / kBlock; }
__device__ __forceinline__ int tiles_of(int rows) { return (rows + kTileRows - 1) / kTileRows; }

// a / b for 0 <= a < 2^24, 0 < b < 2^24 (the quotient by floats is off by one at most):
// the planning is a chain of these, and the compiler's integer division is a longer one.
__device__ __forceinline__ int small_div(int a, int b) {
  int q = (int)__fdividef((float)a, (float)b);
  const int r = a - q * b;
  return q + (r >= b ? 1 : 0) - (r < 0 ? 1 : 0);
}
__device__ __forceinline__ int ceil_div(int a, int b) { return small_div(a + b - 1, b); }

__device__ __noinline__ bool find_item(const PrefixParams& p, const Bars& bars, const GroupPlan* plan, int i,
                                       Item& it) {
  if (i >= bars.total) return false;
  int lo = 0, hi = p.a.groups;                          // the last group whose first item is <= i
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (plan[mid].first <= i) lo = mid;
    else hi = mid;
  }
  const GroupPlan g = plan[lo];
  const int u = small_div(i - g.first, g.splits), split = i - g.first - u * g.splits;
  it.tok0 = g.tok0;
  it.table = g.table;
  it.h = small_div(u, tiles_of(g.rows));
  it.row0 = (u - it.h * tiles_of(g.rows)) * kTileRows;
  it.rows = min(kTileRows, g.rows - it.row0);
  it.tokens = g.pages * p.a.page_len;
  it.ja = split * bars.chunk;
  it.jb = min((it.tokens + kBlock - 1) / kBlock, it.ja + bars.chunk);
  return true;
}

// Every CTA makes the plan for itself (warps 0, 2 and 3): each group's shared pages and
// rows, then the length of a block range.  With c blocks per range the launch takes
// about ceil(items / CTAs) * (c + 1.5) block times (an item's start and end cost about
// one and a half blocks); lane k tries ranges of ceil(longest / (k + 1)) blocks.
__device__ __forceinline__ void plan_groups(const PrefixParams& p, GroupPlan* plan, int w) {
  const SharedAttnParams& a = p.a;
  for (int g = w; g < a.groups; g += 3) {
    int lead;
    const int pages = group_shared_pages(a, g, &lead);
    const int b0 = a.group_indptr[g], b1 = a.group_indptr[g + 1];
    const int tok0 = a.qo_indptr[b0], rows = (a.qo_indptr[b1] - tok0) * a.g;
    if ((threadIdx.x & 31) == 0)
      plan[g] = GroupPlan{rows > 0 ? pages : 0, rows, tok0, rows > 0 ? a.page_indptr[lead] : 0, 0, 0};
  }
}

__device__ __forceinline__ void plan_ranges(const PrefixParams& p, Bars& bars, GroupPlan* plan) {
  const SharedAttnParams& a = p.a;
  const int lane = threadIdx.x & 31, ctas = gridDim.x;
  int longest = 1;
  for (int g = lane; g < a.groups; g += 32) longest = max(longest, blocks_of(plan[g].pages, a.page_len));
  longest = __reduce_max_sync(0xffffffffu, longest);
  const int c = ceil_div(longest, lane + 1);
  int items = 0;
  for (int g = 0; g < a.groups; ++g)
    items += tiles_of(plan[g].rows) * a.Hkv * ceil_div(blocks_of(plan[g].pages, a.page_len), c);
  unsigned cost = 0xffffffffu;
  if (lane == 0 || (lane < longest && items <= p.max_items)) cost = (unsigned)ceil_div(items, ctas) * (2 * c + 3);
  const unsigned win = __reduce_min_sync(0xffffffffu, cost);
  // equal costs: the longer ranges (fewer parts)
  const int chunk = __reduce_max_sync(0xffffffffu, cost == win ? c : 0);
  int run = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    const int g = g0 + lane;
    int n = 0, splits = 0;
    if (g < a.groups) {
      splits = ceil_div(blocks_of(plan[g].pages, a.page_len), chunk);
      n = tiles_of(plan[g].rows) * a.Hkv * splits;
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (g < a.groups) {
      plan[g].splits = splits;
      plan[g].first = run + incl - n;
      if (blockIdx.x == 0) p.plan[g] = plan[g];
    }
    run += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) {
    bars.chunk = chunk;
    bars.total = min(run, p.max_items);
  }
  __syncwarp();
  if (lane == 0) find_item(p, bars, plan, blockIdx.x, bars.first);
}

// Ring positions of block i's K and V among n blocks, in load order.  Two row tiles use
// every block at once: K0 V0 K1 V1 ..; two block streams start with both streams' keys:
// K0 K1 V0 K2 V1 K3 ..
__device__ __forceinline__ int ring_k(bool two, int i) { return two ? 2 * i : i < 2 ? i : 2 * i - 1; }
__device__ __forceinline__ int ring_v(bool two, int i, int n) { return two ? 2 * i + 1 : i < n - 1 ? 2 * i + 2 : 2 * n - 1; }

__device__ __forceinline__ void bar_sync(int id, int count) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(count) : "memory");
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_attn_kernel(const PrefixParams p, const __grid_constant__ CUtensorMap kv_map) {
  using S = Shape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  Bars& bars = *reinterpret_cast<Bars*>(smem + S::kOffBars);
  const SharedAttnParams& a = p.a;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  GroupPlan* plan = a.groups <= kPlanSmem ? bars.plan : p.cta_plan + (int64_t)blockIdx.x * a.groups;

  if (threadIdx.x == 0) {
    mbar_init(&bars.q_ready, 8);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.s_full[t], 1);
      mbar_init(&bars.p_full[t], 4);
    }
    for (int s = 0; s < S::kSlots; ++s) {
      mbar_init(&bars.full[s], 1);
      mbar_init(&bars.empty[s], 1);
    }
    mbar_init(&bars.o_full, 1);
    mbar_init(&bars.drain, 1);
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
  if (warp < 4) {
    pdl_wait();
    pdl_trigger();                                      // the second kernel's own part needs nothing from this one
  }
  if (warp == 0 || warp == 2 || warp == 3) {
    plan_groups(p, plan, warp == 0 ? 0 : warp - 1);
    bar_sync(1, 96);
    if (warp == 2) plan_ranges(p, bars, plan);
  }

  if (warp >= 4) {
    // ------------------------------------------------------------ softmax
    const int t = (warp - 4) >> 2, quarter = warp & 3;
    const int r_local = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tm = tmem + lane_base + kColS + 128 * t, o_tm = tmem + lane_base + kColO + D * t;
    bool ok = true;
    int steps = 0, items = 0;
    // The first round is a rehearsal, while the plan is made: one pass of the block
    // code over whatever the TMEM holds, with nothing waited for, signalled or kept.
    // It brings the loop's instructions (some 10 KB) into the SM's caches, which cost the
    // first real block about 5000 cycles otherwise, twice a later block's time.
    bool rehearse = true;
    Item it;
    it.rows = it.tokens = it.ja = it.row0 = it.h = it.tok0 = 0;
    it.jb = 1;
    for (int i = blockIdx.x;;) {
      const bool two = it.rows > 128;
      const int n = it.jb - it.ja, count = rehearse ? 1 : two ? n : (n + 1 - t) / 2;
      const int my0 = two ? 128 * t : 0;                // this stream's first row of the tile
      if (!rehearse) {
        if (two || t == 0) {
          // the warp's 32 query rows into the swizzled A operand, two (D = 128) or four
          // rows per load instruction; the previous item's products have all completed
          constexpr int kChunks = D / 8, kPer = 32 / kChunks, kLoads = 32 / kPer;
          const int chunk = lane % kChunks;
          const uint32_t qb = smem_u32(smem + S::kOffQ + (two ? t : 0) * S::kSlotBytes) + (chunk / 8) * S::kQHalfBytes;
          const uint16_t* q = (const uint16_t*)a.q + ((int64_t)it.tok0 * a.Hq + it.h * a.g) * D + chunk * 8;
          for (int k0 = 0; k0 < kLoads; k0 += 8) {
            uint4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int r = quarter * 32 + (k0 + k) * kPer + lane / kChunks, R = it.row0 + my0 + r;
              const int tk = p.div_g.div(R);
              v[k] = make_uint4(0, 0, 0, 0);
              if (my0 + r < it.rows) v[k] = __ldg((const uint4*)(q + ((int64_t)tk * a.Hq + (R - tk * a.g)) * D));
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int r = quarter * 32 + (k0 + k) * kPer + lane / kChunks;
              st_shared_v4(qb + (uint32_t)r * 128u + (uint32_t)(((chunk & 7) ^ (r & 7)) << 4), v[k].x, v[k].y, v[k].z,
                           v[k].w);
            }
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_ready);
      }
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
        const int left = it.tokens - (it.ja + (two ? x : 2 * x + t)) * kBlock;
        if (left < kBlock) {
#pragma unroll
          for (int c = 0; c < kBlock; ++c)
            if (c >= left) s[c / 64][c % 64] = __float_as_uint(-INFINITY);
        }
        float x0 = -INFINITY, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
#pragma unroll
        for (int c = 0; c < kBlock; c += 8) {
          x0 = fmax3(x0, __uint_as_float(s[c / 64][c % 64 + 0]), __uint_as_float(s[c / 64][c % 64 + 1]));
          x1 = fmax3(x1, __uint_as_float(s[c / 64][c % 64 + 2]), __uint_as_float(s[c / 64][c % 64 + 3]));
          x2 = fmax3(x2, __uint_as_float(s[c / 64][c % 64 + 4]), __uint_as_float(s[c / 64][c % 64 + 5]));
          x3 = fmax3(x3, __uint_as_float(s[c / 64][c % 64 + 6]), __uint_as_float(s[c / 64][c % 64 + 7]));
        }
        const float top = fmax3(x0, x1, fmaxf(x2, x3)) * p.scale_log2;
        const bool need = top > m + kRescale;
        float alpha = 1.0f;
        if (need) {
          alpha = m == -INFINITY ? 0.0f : fast_exp2(m - top);
          l *= alpha;
          m = top;
        }
        const float sub = m == -INFINITY ? 0.0f : m;
        const uint64_t sc2 = f2(p.scale_log2, p.scale_log2), nm2 = f2(-sub, -sub);
        uint64_t l0 = f2(0.0f, 0.0f), l1 = l0;
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
        }
        float a0, a1;
        f2_split(fadd2(l0, l1), a0, a1);
        l += a0 + a1;
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
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (!rehearse) {
          if (lane == 0) mbar_arrive(&bars.p_full[t]);
          ++steps;
        }
      }
      if (!ok) {
        if (lane == 0) give_up(p, 71);
        break;
      }
      if (rehearse) {
        rehearse = false;
        pdl_wait();
        pdl_trigger();
        __syncthreads();                                // the plan is complete
        if (i >= bars.total) break;
        it = bars.first;
        continue;
      }
      ok = __all_sync(0xffffffffu, mbar_wait(&bars.o_full, items & 1, p.wait_limit));
      if (!ok) {
        if (lane == 0) give_up(p, 72);
        break;
      }
      tc_fence_after();
      // the part: O as [column quad][row] so that a warp stores 512 contiguous bytes
      float* part = p.parts + (int64_t)i * S::kPartFloats + t * (S::kPartFloats / 2);
      const bool valid = my0 + r_local < it.rows;
#pragma unroll 1
      for (int cb = 0; cb < D / 32; ++cb) {
        uint32_t o[32];
        tmem_ld32(o_tm + 32 * cb, o);
        tmem_ld_wait();
        if (valid) {
#pragma unroll
          for (int qd = 0; qd < 8; ++qd)
            *(float4*)(part + ((cb * 8 + qd) * 128 + r_local) * 4) =
                make_float4(__uint_as_float(o[4 * qd]), __uint_as_float(o[4 * qd + 1]),
                            __uint_as_float(o[4 * qd + 2]), __uint_as_float(o[4 * qd + 3]));
        }
      }
      tc_fence_before();
      if (valid) {
        part[128 * D + r_local] = m;
        part[128 * D + 128 + r_local] = l;
      }
      ++items;
      i += gridDim.x;
      if (!find_item(p, bars, plan, i, it)) break;
    }
  } else {
    __syncthreads();                                    // the plan is complete
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer
      // Lane r brings the r-th copy of a block.  The page of load x + 4 is fetched while
      // load x is issued (unrolled by four, so that no register that a fetch is still
      // filling is moved).
      const int copies = kBlock / p.copy_tokens;
      bool ok = true;
      int pushed = 0;                                   // copies into the ring so far
      Item it = bars.first;
      for (int i = blockIdx.x; ok && i < bars.total;) {
        const bool two = it.rows > 128;
        const int n = it.jb - it.ja;
        const int32_t* table = a.page_indices + it.table;
        // the x-th load: K or V, and this lane's token of it
        auto what = [&](int x, bool& is_v, int& tok) {
          int j;
          if (two) {                                    // K0 V0 K1 V1 ..
            is_v = x & 1;
            j = x >> 1;
          } else if (x < min(2, n)) {                   // K0 K1 V0 K2 V1 .. , the last two V
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
          if (page < 0 || page >= a.max_pages) page = a.max_pages;  // past the pool: zero fill
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
        i += gridDim.x;
        if (!find_item(p, bars, plan, i, it)) break;
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
        int base = 0, items = 0, steps[2] = {0, 0};     // ring positions before this item; items and blocks done
        auto wait = [&](uint64_t* bar, int parity, int code) {
          ok = ok && mbar_wait(bar, parity & 1, p.wait_limit);
          if (!ok) give_up(p, code);
          tc_fence_after();
          return ok;
        };
        Item it = bars.first;
        for (int i = blockIdx.x; ok && i < bars.total;) {
          const bool two = it.rows > 128;
          const int n = it.jb - it.ja;
          const int count[2] = {two ? n : (n + 1) / 2, two ? n : n / 2};
          if (!wait(&bars.q_ready, items, 61)) break;
          // step 2 x + t: O += P V of stream t's block x - 1, then S = Q K^T of its block x
          for (int st = 0; ok && st < 2 * (count[0] + 1); ++st) {
            const int t = st & 1, x = st >> 1;
            if (x > count[t]) continue;
            if (x > 0) {
              const int pos = base + ring_v(two, two ? x - 1 : 2 * (x - 1) + t, n), slot = pos % S::kSlots;
              if (!wait(&bars.full[slot], pos / S::kSlots, 63) || !wait(&bars.p_full[t], steps[t], 64)) break;
              ++steps[t];
              const uint64_t vd = v0 + (uint64_t)((slot * S::kSlotBytes) >> 4);
#pragma unroll
              for (int k = 0; k < kRuns; ++k)
                mma_bf16_ts(tmem + kColO + D * t, tmem + kColS + 128 * t + 8 * k,
                            vd + (uint64_t)((k * S::kRunBytes) >> 4), id_pv, (x > 1 || k > 0) ? 1u : 0u);
              if (!two || t == 1) mma_commit(&bars.empty[slot]);
            }
            if (x < count[t]) {
              const int pos = base + ring_k(two, two ? x : 2 * x + t), slot = pos % S::kSlots;
              if (!wait(&bars.full[slot], pos / S::kSlots, 65)) break;
              const uint64_t qd = q0 + (uint64_t)((two ? t * S::kSlotBytes : 0u) >> 4);
              const uint64_t kd = k0 + (uint64_t)((slot * S::kSlotBytes) >> 4);
#pragma unroll
              for (int k = 0; k < D / 16; ++k)
                mma_bf16_ss(tmem + kColS + 128 * t, qd + (uint64_t)(((k / 4) * S::kQHalfBytes + (k % 4) * 32) >> 4),
                            kd + (uint64_t)(((k / 4) * 1024 + (k % 4) * 32) >> 4), id_qk, k > 0);
              mma_commit(&bars.s_full[t]);
              if (!two || t == 1) mma_commit(&bars.empty[slot]);
              issued = true;
            }
          }
          if (ok) mma_commit(&bars.o_full);
          base += 2 * n;
          ++items;
          i += gridDim.x;
          if (!find_item(p, bars, plan, i, it)) break;
        }
        if (issued) {
          mma_commit(&bars.drain);
          mbar_wait(&bars.drain, 0);
        }
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// --------------------------------------------------------------- own columns
constexpr int kOwnThreads = 128;
constexpr int kOwnTile = 32;              // tokens staged at a time
constexpr int kOwnStages = 3;
constexpr int kMaxOwnSplits = 32;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;                         // 0: the 16 bytes are zeroed
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull; }

// Which of own columns c0 .. c0 + 63 row `node` sees (bit i: column c0 + i): those
// before `prefix`, then tree slots by the row's mask, or up to its own without masks.
__device__ __forceinline__ uint64_t seen_columns(const SharedAttnParams& a, const uint64_t* mask, int node, int c0,
                                                 int prefix, int len) {
  uint64_t v = low_bits(min(prefix, len) - c0);
  const int first = max(prefix, c0);                    // first tree column of the 64
  if (first < min(len, c0 + 64)) {
    const int slot = first - prefix;
    uint64_t bits;
    if (!a.mask_bits) {
      bits = low_bits(node - slot + 1);
    } else {
      const int w = slot >> 6, sh = slot & 63;
      const uint64_t lo = w < a.mask_words ? __ldg(mask + w) : 0ull;
      const uint64_t hi = sh && w + 1 < a.mask_words ? __ldg(mask + w + 1) : 0ull;
      bits = sh ? (lo >> sh) | (hi << (64 - sh)) : lo;
    }
    v |= (bits & low_bits(min(len, c0 + 64) - first)) << (first - c0);
  }
  return v;
}

// Joins rows 0 .. n - 1 (request rows row0 ..) of request b and KV head h: their own
// parts, and the shared parts of their group.  Own part k of row r: O at own_o + k *
// o_part + r * o_row, (m, l) at own_ml + k * ml_part + r * ml_row.  `w` and `lw` hold
// [kMaxParts][ROWS] floats.  First every part's m and l come in at once, then a thread
// per row turns them into weights e^(m - M) / L, then each thread sums one column quad of
// one row: four rows and eight quads per warp, so that both the parts ([quad][row]) and
// the output are touched in 64-byte pieces.
constexpr int kMaxParts = 2 * kMaxSplits + kMaxOwnSplits;

template <int D, int ROWS>
__device__ __forceinline__ void join_rows(const PrefixParams& p, const GroupPlan& g, int gi, int b, int h, int row0,
                                          int n, const float* own_o, int64_t o_part, int64_t o_row,
                                          const float2* own_ml, int64_t ml_part, int64_t ml_row, int own_parts,
                                          float* w, float* lw) {
  const SharedAttnParams& a = p.a;
  constexpr int kPart = Shape<D>::kPartFloats, kHalf = kPart / 2;
  const int tok0 = a.qo_indptr[b];
  const int in_group = (tok0 - a.qo_indptr[a.group_indptr[gi]]) * a.g + row0;
  const int tiles = (g.rows + kTileRows - 1) / kTileRows;
  // row r's shared part k: stream k & 1 of range k / 2 where two block streams shared
  // the rows, else its row half's stream of range k
  const float* first = p.parts + ((int64_t)g.first + (int64_t)h * tiles * g.splits) * kPart;
  auto part_of = [&](int r, int k, int& shared) -> const float* {
    const int rg = in_group + r, tile = rg / kTileRows, in = rg % kTileRows;
    const bool two = g.rows - tile * kTileRows > 128;
    shared = two ? g.splits : 2 * g.splits;
    return first + (int64_t)tile * g.splits * kPart + (two ? (int64_t)k * kPart + (in >> 7) * kHalf : (int64_t)k * kHalf) +
           (in & 127) * 4;
  };
  const int most = 2 * g.splits + own_parts;
#pragma unroll 4
  for (int e = threadIdx.x; e < most * ROWS; e += kOwnThreads) {
    const int k = e / ROWS, r = e % ROWS;
    float m = -INFINITY, l = 0.0f;
    if (r < n) {
      int shared;
      const float* s = part_of(r, k, shared);
      if (k < shared) {
        const float* ml = s - ((in_group + r) % 128) * 4 + 128 * D + (in_group + r) % 128;
        m = __ldcg(ml);
        l = __ldcg(ml + 128);
      } else if (k - shared < own_parts) {
        const float2 x = own_ml[(k - shared) * ml_part + r * ml_row];
        m = x.x;
        l = x.y;
      }
    }
    w[e] = m;
    lw[e] = l;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < ROWS; r += kOwnThreads) {
    float M = -INFINITY, L = 0.0f;
    for (int k = 0; k < most; ++k) M = fmaxf(M, w[k * ROWS + r]);
    const float base = M == -INFINITY ? 0.0f : M;
    for (int k = 0; k < most; ++k) {
      const float x = fast_exp2(w[k * ROWS + r] - base);
      L = fmaf(x, lw[k * ROWS + r], L);
      w[k * ROWS + r] = x;
    }
    lw[r] = L > 0.0f ? 1.0f / L : L == L ? 0.0f : L;    // nothing seen: 0
  }
  __syncthreads();
  const int units = (n + 3) / 4 * D;
  for (int idx = threadIdx.x; idx < units; idx += kOwnThreads) {
    const int lo = idx & 31, hi = idx >> 5;
    const int r = (hi / (D / 32)) * 4 + (lo & 3), quad = (hi % (D / 32)) * 8 + (lo >> 2);
    if (r >= n) continue;
    float o0 = 0.0f, o1 = 0.0f, o2 = 0.0f, o3 = 0.0f;
    int shared;
    const float* s = part_of(r, 0, shared) + quad * 512;
    const int64_t step = shared == g.splits ? kPart : kHalf;
    for (int k0 = 0; k0 < shared; k0 += 8) {
      float4 v[8];                                      // eight loads in flight
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (k0 + u < shared) v[u] = __ldcg((const float4*)(s + (k0 + u) * step));
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float x = k0 + u < shared ? w[(k0 + u) * ROWS + r] : 0.0f;
        if (x != 0.0f) {                                // a part of no columns has no O
          o0 = fmaf(x, v[u].x, o0);
          o1 = fmaf(x, v[u].y, o1);
          o2 = fmaf(x, v[u].z, o2);
          o3 = fmaf(x, v[u].w, o3);
        }
      }
    }
#pragma unroll 2
    for (int k = 0; k < own_parts; ++k) {
      const float x = w[(shared + k) * ROWS + r];
      if (x != 0.0f) {
        const float4 v = *(const float4*)(own_o + k * o_part + r * o_row + quad * 4);
        o0 = fmaf(x, v.x, o0);
        o1 = fmaf(x, v.y, o1);
        o2 = fmaf(x, v.z, o2);
        o3 = fmaf(x, v.w, o3);
      }
    }
    const float inv = lw[r];
    const int R = row0 + r, tk = p.div_g.div(R);
    *(uint2*)((uint16_t*)a.out + ((int64_t)(tok0 + tk) * a.Hq + h * a.g + R - tk * a.g) * D + quad * 4) =
        make_uint2(pack_bf16x2(o0 * inv, o1 * inv), pack_bf16x2(o2 * inv, o3 * inv));
  }
}

// Shared memory of own_attn_kernel: the stages, or O and the weights of the join.
template <int D, int WR>
constexpr size_t own_smem() {
  constexpr int WT = WR == 1 ? 2 : 1, kRows = 16 * WR;
  constexpr size_t stages = (size_t)kOwnStages * 2 * kOwnTile * D * 2;
  constexpr size_t join = ((size_t)WT * kRows * D + 2 * (2 * kMaxSplits + WT) * kRows) * 4;
  return stages > join ? stages : join;
}

// 16 WR rows of a request per CTA.  The four warps are WR row groups x WT token groups x
// WD halves of the output dimensions: with few rows the tokens and dimensions are split
// instead (the scores are then computed twice, which costs nothing next to the loads),
// so that a thread's O stays at 32 registers and four CTAs fit an SM.
template <int D, int WR>
__global__ void __launch_bounds__(kOwnThreads, WR == 4 ? 3 : 4) own_attn_kernel(const PrefixParams p) {
  constexpr int WD = WR == 4 ? 1 : 2, WT = 4 / (WR * WD), kRows = 16 * WR, kChunks = D / 8, kRowBytes = D * 2;
  constexpr int NC = kOwnTile / WT / 16;                // 16-token chunks of a warp
  constexpr int DW = D / WD;                            // its output dimensions
  constexpr uint32_t kTileBytes = kOwnTile * kRowBytes; // K or V
  extern __shared__ __align__(16) uint8_t stage[];
  __shared__ float2 ml[WT][kRows];
  const SharedAttnParams& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  const int wr = warp % WR, wt = warp / WR % WT, wd = warp / (WR * WT);
  const int b = blockIdx.x / p.request_tiles, row0 = (blockIdx.x - b * p.request_tiles) * kRows, h = blockIdx.y;
  const int tok0 = a.qo_indptr[b], n_tok = a.qo_indptr[b + 1] - tok0, total_rows = n_tok * a.g;
  pdl_trigger();
  if (row0 >= total_rows) {
    pdl_wait();                                         // no CTA ends before the first kernel has: what follows may
    return;                                             // wait for this one alone
  }
  const int rows = min(kRows, total_rows - row0);
  const int gi = group_of(a, b);
  const int shared = group_shared_pages(a, gi);
  const int32_t* table = a.page_indices + a.page_indptr[b] + shared;
  const int len = max(0, kv_tokens(a, b) - shared * a.page_len), prefix = len - n_tok;
  const int n_tiles = (len + kOwnTile - 1) / kOwnTile;
  const int j0 = (int)((int64_t)n_tiles * blockIdx.z / p.own_splits);
  const int j1 = (int)((int64_t)n_tiles * (blockIdx.z + 1) / p.own_splits);
  const uint32_t smem0 = smem_u32(stage);
  const int64_t tok_elems = (int64_t)a.Hkv * D;
  const uint16_t* kv = (const uint16_t*)a.kv + (int64_t)h * D;

  // Where 16-token runs 32 w .. 32 w + 31 start (lane i: run 32 w + i), in elements of the
  // pool's head h; -1: not in the pool.
  auto window = [&](int w) -> int64_t {
    const int tok = (32 * w + lane) * 16;
    if (tok >= len) return -1;
    const int pg = p.page_of(tok), page = __ldg(table + pg);
    if (page < 0 || page >= a.max_pages) return -1;
    return ((int64_t)page * 2 * a.page_len + (tok - pg * a.page_len)) * tok_elems;
  };
  constexpr int kTilesPerWindow = 32 * 16 / kOwnTile;
  int win = j0 / kTilesPerWindow;
  int64_t at = window(win), at_next = window(win + 1);
  auto load_tile = [&](int j) {
    if (j / kTilesPerWindow != win) {
      ++win;
      at = at_next;
      at_next = window(win + 1);
    }
    const uint32_t buf = smem0 + (j % kOwnStages) * 2 * kTileBytes;
#pragma unroll
    for (int e0 = 0; e0 < kOwnTile * kChunks; e0 += kOwnThreads) {
      const int e = e0 + threadIdx.x, t = e / kChunks, c = e % kChunks;
      const int64_t run = __shfl_sync(0xffffffffu, at, (j * (kOwnTile / 16) + t / 16) & 31);
      const bool valid = run >= 0 && j * kOwnTile + t < len;
      const uint16_t* src = valid ? kv + run + (t & 15) * tok_elems + c * 8 : kv;
      const uint32_t dst = buf + t * kRowBytes + ((c ^ (t & 7)) << 4);
      cp_async16(dst, src, valid);
      cp_async16(dst + kTileBytes, valid ? src + a.page_len * tok_elems : src, valid);
    }
    cp_async_commit();
  };
  static_assert(kOwnThreads / kChunks <= 16, "the lanes of a warp load one run at a time");

  for (int s = 0; s < kOwnStages - 1; ++s) {
    if (j0 + s < j1) load_tile(j0 + s);
    else cp_async_commit();
  }
  // the warp's 16 query rows as A fragments; rows past the request's are zero
  uint32_t qa[D / 16][4];
  int node[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = wr * 16 + gq + 8 * i, R = row0 + r;
    const bool valid = r < rows;
    node[i] = valid ? p.div_g.div(R) : 0;
    const uint16_t* q =
        (const uint16_t*)a.q + ((int64_t)(tok0 + node[i]) * a.Hq + h * a.g + (valid ? R - node[i] * a.g : 0)) * D + 2 * tq;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qa[k][i] = valid ? __ldg((const uint32_t*)(q + 16 * k)) : 0u;
      qa[k][2 + i] = valid ? __ldg((const uint32_t*)(q + 16 * k + 8)) : 0u;
    }
  }
  float o[DW / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < DW / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  const int mi = lane >> 3, rr = lane & 7;

  for (int j = j0; j < j1; ++j) {
    if (j + kOwnStages - 1 < j1) load_tile(j + kOwnStages - 1);
    else cp_async_commit();
    cp_async_wait<kOwnStages - 1>();
    __syncthreads();
    const uint32_t kb = smem0 + (j % kOwnStages) * 2 * kTileBytes, vb = kb + kTileBytes;
    const int c0 = j * kOwnTile, t0 = wt * (kOwnTile / WT);
    float s[NC][2][4];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c][e >> 2][e & 3] = 0.0f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int t = t0 + 16 * c + rr + 8 * (mi >> 1);
        uint32_t r0, r1, r2, r3;
        ldmatrix_x4(kb + t * kRowBytes + (((2 * k + (mi & 1)) ^ (t & 7)) << 4), r0, r1, r2, r3);
        mma_m16n8k16(s[c][0], qa[k], r0, r1);
        mma_m16n8k16(s[c][1], qa[k], r2, r3);
      }
    const bool masked = c0 + kOwnTile > prefix;         // tree slots or the end in this tile
    uint32_t seen[2] = {~0u, ~0u};
    if (masked) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        seen[i] = seen_columns(a, a.mask_bits ? a.mask_bits + (int64_t)(tok0 + node[i]) * a.mask_words : nullptr,
                               node[i], c0, prefix, len);
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float& x = s[c][e >> 2][e & 3];
        const int i = (e >> 1) & 1, col = t0 + 16 * c + 8 * (e >> 2) + 2 * tq + (e & 1);
        x = (seen[i] >> col) & 1u ? x * p.scale_log2 : -INFINITY;
        top[i] = fmaxf(top[i], x);
      }
    float keep[2], sub[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      const float nm = fmaxf(m[i], top[i]);
      sub[i] = nm == -INFINITY ? 0.0f : nm;
      keep[i] = fast_exp2(m[i] - sub[i]);
      m[i] = nm;
      l[i] *= keep[i];
    }
#pragma unroll
    for (int i = 0; i < DW / 8; ++i) {
      o[i][0] *= keep[0];
      o[i][1] *= keep[0];
      o[i][2] *= keep[1];
      o[i][3] *= keep[1];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float& x = s[c][e >> 2][e & 3];
        x = fast_exp2(x - sub[(e >> 1) & 1]);
        l[(e >> 1) & 1] += x;
      }
    // Values that 0 * v does not cancel, in a tile where rows see different slots: only
    // the rows that see them may take them.
    bool odd = false;
    if (masked && n_tok > 1) {
      for (int e = threadIdx.x; e < kOwnTile * kChunks; e += kOwnThreads) {
        const uint4 v = ld_shared_v4(vb + e * 16);
        auto bad = [](uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; };
        odd |= bad(v.x) || bad(v.y) || bad(v.z) || bad(v.w);
      }
      odd = __syncthreads_or(odd);
    }
    if (!odd) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint32_t pa[4] = {pack_bf16x2(s[c][0][0], s[c][0][1]), pack_bf16x2(s[c][0][2], s[c][0][3]),
                                pack_bf16x2(s[c][1][0], s[c][1][1]), pack_bf16x2(s[c][1][2], s[c][1][3])};
#pragma unroll
        for (int d = 0; d < DW / 16; ++d) {
          const int t = t0 + 16 * c + rr + 8 * (mi & 1), ch = wd * (DW / 8) + 2 * d + (mi >> 1);
          uint32_t r0, r1, r2, r3;
          ldmatrix_x4_trans(vb + t * kRowBytes + ((ch ^ (t & 7)) << 4), r0, r1, r2, r3);
          mma_m16n8k16(o[2 * d], pa, r0, r1);
          mma_m16n8k16(o[2 * d + 1], pa, r2, r3);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int u = 0; u < 16; ++u) {                  // token u of the 16: its lane of the quad, its element
          const float p0 = __shfl_sync(0xffffffffu, s[c][u >> 3][u & 1], (lane & ~3) | ((u & 7) >> 1));
          const float p1 = __shfl_sync(0xffffffffu, s[c][u >> 3][2 + (u & 1)], (lane & ~3) | ((u & 7) >> 1));
          const int t = t0 + 16 * c + u;
#pragma unroll
          for (int d = 0; d < DW / 8; ++d) {
            uint32_t w;
            asm volatile("ld.shared.b32 %0, [%1];"
                         : "=r"(w)
                         : "r"(vb + t * kRowBytes + (((wd * (DW / 8) + d) ^ (t & 7)) << 4) + 4 * tq));
            const float v0 = bf16_bits_to_float(w & 0xffffu), v1 = bf16_bits_to_float(w >> 16);
            if (p0 != 0.0f) {
              o[d][0] = fmaf(p0, v0, o[d][0]);
              o[d][1] = fmaf(p0, v1, o[d][1]);
            }
            if (p1 != 0.0f) {
              o[d][2] = fmaf(p1, v0, o[d][2]);
              o[d][3] = fmaf(p1, v1, o[d][3]);
            }
          }
        }
    }
    __syncthreads();                                    // the stage may be loaded again
  }
  cp_async_wait<0>();
  __syncthreads();
  float* os = (float*)stage;                            // [WT][rows][D]
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    const int r = wr * 16 + gq + 8 * i;
    if (tq == 0 && wd == 0) ml[wt][r] = make_float2(m[i], l[i]);
#pragma unroll
    for (int d = 0; d < DW / 8; ++d)
      *(float2*)(os + (wt * kRows + r) * D + wd * DW + 8 * d + 2 * tq) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
  }
  __syncthreads();
  if (p.own_splits > 1) {
    // a slice of the own columns: one part per row for the join kernel
    for (int e = threadIdx.x; e < rows * (D / 4); e += kOwnThreads) {
      const int r = e / (D / 4), quad = e % (D / 4), R = row0 + r, tk = p.div_g.div(R);
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < WT; ++w) M = fmaxf(M, ml[w][r].x);
      const float sub = M == -INFINITY ? 0.0f : M;
      float L = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < WT; ++w) {
        const float f = fast_exp2(ml[w][r].x - sub);
        if (f == 0.0f) continue;
        const float4 v = *(const float4*)(os + (w * kRows + r) * D + quad * 4);
        L = fmaf(f, ml[w][r].y, L);
        acc.x = fmaf(f, v.x, acc.x);
        acc.y = fmaf(f, v.y, acc.y);
        acc.z = fmaf(f, v.z, acc.z);
        acc.w = fmaf(f, v.w, acc.w);
      }
      const int64_t row = (int64_t)(tok0 + tk) * a.Hq + h * a.g + R - tk * a.g, part = row * p.own_splits + blockIdx.z;
      *(float4*)(p.own_o + part * D + quad * 4) = acc;
      if (quad == 0) p.own_ml[part] = make_float2(M, L);
    }
    pdl_wait();
    return;
  }
  // the weights go behind O in the stage
  constexpr int kOFloats = WT * kRows * D, kWeights = (2 * kMaxSplits + WT) * kRows;
  static_assert((kOFloats + 2 * kWeights) * 4 <= own_smem<D, WR>(), "the join's arrays");
  pdl_wait();                                           // the shared parts are complete
  join_rows<D, kRows>(p, p.plan[gi], gi, b, h, row0, rows, os, kRows * D, D, &ml[0][0], kRows, 1, WT, os + kOFloats,
                      os + kOFloats + kWeights);
}

// After own_attn_kernel with several slices: one CTA per (request row, KV head) joins a
// token's heads.
template <int D>
__global__ void __launch_bounds__(kOwnThreads) join_parts_kernel(const PrefixParams p) {
  const SharedAttnParams& a = p.a;
  constexpr int kRows = 16;
  __shared__ float w[kMaxParts * kRows], lw[kMaxParts * kRows];
  pdl_trigger();
  pdl_wait();
  const int tok = blockIdx.x, h = blockIdx.y;
  if (tok >= a.qo_indptr[a.batch]) return;
  int lo = 0, hi = a.batch;                             // the request of the token
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.qo_indptr[mid] <= tok) lo = mid;
    else hi = mid;
  }
  const int gi = group_of(a, lo), node = tok - a.qo_indptr[lo];
  for (int r0 = 0; r0 < a.g; r0 += kRows) {
    const int64_t row = (int64_t)tok * a.Hq + h * a.g + r0;
    join_rows<D, kRows>(p, p.plan[gi], gi, lo, h, node * a.g + r0, min(kRows, a.g - r0), p.own_o + row * p.own_splits * D,
                        D, (int64_t)p.own_splits * D, p.own_ml + row * p.own_splits, 1, p.own_splits, p.own_splits, w,
                        lw);
    __syncthreads();
  }
}

struct PrefixPlan {
  int own_rows, request_tiles, own_splits, max_items, ctas;
  size_t plan, cta_plan, parts, own_ml, own_o, bytes;
};

int sm_count() {
  static int count = 0;
  if (!count) {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
      count = n;
  }
  return count ? count : 148;
}

PrefixPlan plan_prefix(int batch, int groups, int total_q, int max_qo_len, int max_kv_len, int max_own_len, int Hq,
                       int Hkv, int D) {
  PrefixPlan f;
  const int g = Hq / Hkv;
  const int64_t rows = (int64_t)max_qo_len * g;
  f.own_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  f.request_tiles = (int)((rows + f.own_rows - 1) / f.own_rows);
  f.ctas = sm_count();
  // own columns: about four CTAs per SM, each with four tiles at least
  const int64_t ctas = (int64_t)batch * f.request_tiles * Hkv;
  const int own = max_own_len > 0 ? max_own_len : max_kv_len;
  f.own_splits = (int)std::max<int64_t>(1, std::min<int64_t>({4ll * f.ctas / std::max<int64_t>(ctas, 1),
                                                              (own + 4 * kOwnTile - 1) / (4 * kOwnTile),
                                                              kMaxOwnSplits}));
  const int64_t units = (((int64_t)total_q * g + kTileRows - 1) / kTileRows + groups) * Hkv;
  f.max_items = (int)std::min<int64_t>(units + 2 * f.ctas, 1 << 30);
  const int part = D == 128 ? Shape<128>::kPartFloats : Shape<64>::kPartFloats;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at = align_up(at + n, 256);
    return o;
  };
  f.plan = take(sizeof(GroupPlan) * groups);
  f.cta_plan = take(groups > kPlanSmem ? sizeof(GroupPlan) * groups * f.ctas : 0);
  f.parts = take((size_t)f.max_items * part * sizeof(float));
  const size_t own_parts = f.own_splits > 1 ? (size_t)total_q * Hq * f.own_splits : 0;
  f.own_ml = take(own_parts * sizeof(float2));
  f.own_o = take(own_parts * D * sizeof(float));
  f.bytes = at;
  return f;
}

template <int D, int WR>
int launch_own(const PrefixParams& p, cudaStream_t stream) {
  constexpr size_t smem = own_smem<D, WR>();
  if (int rc = ensure_smem_attr((const void*)own_attn_kernel<D, WR>, smem)) return rc;
  PTS_CUDA_TRY(launch_pdl(own_attn_kernel<D, WR>, dim3(p.a.batch * p.request_tiles, p.a.Hkv, p.own_splits),
                          dim3(kOwnThreads), smem, stream, p));
  return launch_status("own_attn_kernel");
}

template <int D>
int launch_prefix(const PrefixParams& p, const PrefixPlan& f, int total_q, cudaStream_t stream) {
  const SharedAttnParams& a = p.a;
  CUtensorMap map;
  // (dim of a half, token of a group, head and half, group, 2 page + K/V)
  const cuuint64_t tok = (cuuint64_t)a.Hkv * D * 2;
  const cuuint64_t dims[5] = {64, 8, (cuuint64_t)a.Hkv * (D / 64), (cuuint64_t)a.page_len / 8, (cuuint64_t)a.max_pages * 2};
  const cuuint64_t strides[4] = {tok, 128, 8 * tok, a.page_len * tok};
  const cuuint32_t box[5] = {64, 8, D / 64, (cuuint32_t)p.copy_tokens / 8, 1};
  if (int rc = encode_tiled_bf16_sw128(&map, 5, a.kv, dims, strides, box)) return rc;
  if (int rc = ensure_smem_attr((const void*)prefix_attn_kernel<D>, Shape<D>::kSmem)) return rc;
  PTS_CUDA_TRY(launch_pdl(prefix_attn_kernel<D>, dim3(f.ctas), dim3(kThreads), Shape<D>::kSmem, stream, p, map));
  if (int rc = launch_status("prefix_attn_kernel")) return rc;
  int rc = f.own_rows == 16 ? launch_own<D, 1>(p, stream) : f.own_rows == 32 ? launch_own<D, 2>(p, stream)
                                                                            : launch_own<D, 4>(p, stream);
  if (rc || p.own_splits == 1) return rc;
  PTS_CUDA_TRY(launch_pdl(join_parts_kernel<D>, dim3(total_q, a.Hkv), dim3(kOwnThreads), 0, stream, p));
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
  if ((int64_t)a.batch * ((int64_t)max_qo_len * a.g / 16 + 1) > 2147483647ll)
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
  p.max_items = f.max_items;
  p.parts = (float*)(ws + f.parts);
  p.plan = (GroupPlan*)(ws + f.plan);
  p.cta_plan = (GroupPlan*)(ws + f.cta_plan);
  p.error = error;
  p.wait_limit = wait_limit_cycles();
  p.own_splits = f.own_splits;
  p.request_tiles = f.request_tiles;
  p.own_o = (float*)(ws + f.own_o);
  p.own_ml = (float2*)(ws + f.own_ml);
  return a.D == 128 ? launch_prefix<128>(p, f, total_q, stream) : launch_prefix<64>(p, f, total_q, stream);
}

}  // namespace pts
