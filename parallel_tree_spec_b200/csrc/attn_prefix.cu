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
constexpr int kRun = 16;                  // tokens per TMA copy
constexpr int kTileRows = 256;
constexpr int kThreads = 384;             // warps 0 TMA, 1 MMA, 2-3 plan only, 4-7 and 8-11 softmax
constexpr int kMaxSplits = 64;
constexpr int kPlanSmem = 48;             // groups whose plan fits in shared memory
constexpr float kRescale = 8.0f;          // O is rescaled when the row max grows by more than 2^8
constexpr uint32_t kColS = 0, kColO = 256;

template <int D>
struct Shape {
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kHalfBytes = kBlock * 128;          // 128 rows of 64 bf16
  static constexpr uint32_t kSlotBytes = kHalves * kHalfBytes;  // K or V of a block; Q of a stream
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr uint32_t kOffQ = 0;
  static constexpr uint32_t kOffRing = 2 * kSlotBytes;
  static constexpr uint32_t kOffBars = kOffRing + kSlots * kSlotBytes;
  static constexpr uint32_t kSmem = kOffBars + 1280 + 1024;     // barriers, plan; alignment slack
  static constexpr int kPartFloats = 2 * 128 * (D + 2);         // one item's part
};
static_assert(Shape<128>::kSmem <= 232448 && Shape<64>::kSmem <= 232448, "shared memory above 227 KB");

struct GroupPlan {
  int pages;      // shared pages
  int rows;       // query rows per KV head
  int first;      // first work item
  int splits;     // block ranges per (row tile, KV head)
};

struct __align__(8) Bars {
  uint64_t q_ready;         // both warpgroups: done with the last item, this one's rows stored
  uint64_t full[8], empty[8];
  uint64_t s_full[2], p_full[2];
  uint64_t o_full, drain;
  uint32_t tmem;
  int abort;
  int chunk, total;         // blocks per range, work items
  GroupPlan plan[kPlanSmem];
};
static_assert(sizeof(Bars) <= 1280, "barrier block");

struct PrefixParams {
  SharedAttnParams a;
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
};

__device__ __forceinline__ void give_up(Bars& bars, const PrefixParams& p, int code) {
  *(volatile int*)&bars.abort = 1;
  if (p.error) atomicExch(p.error, code);
}
__device__ __forceinline__ bool gave_up(const Bars& bars) { return *(volatile const int*)&bars.abort != 0; }

__device__ __forceinline__ int blocks_of(int pages, int page_len) { return (pages * page_len + kBlock - 1) / kBlock; }

// One work item.
struct Item {
  int group, h, tile, b0;   // b0: the group's first request with rows
  int tok0, rows, row0;     // rows of the tile: row0 .. of the group's rows per KV head
  int ja, jb, tokens;       // blocks; tokens of the shared columns
};

__device__ __forceinline__ bool find_item(const PrefixParams& p, const Bars& bars, const GroupPlan* plan, int i,
                                          Item& it) {
  if (i >= bars.total) return false;
  int lo = 0, hi = p.a.groups;                          // the last group whose first item is <= i
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (plan[mid].first <= i) lo = mid;
    else hi = mid;
  }
  const GroupPlan g = plan[lo];
  const int tiles = (g.rows + kTileRows - 1) / kTileRows;
  int u = i - g.first;
  const int split = u % g.splits;
  u /= g.splits;
  it.group = lo;
  it.tile = u % tiles;
  it.h = u / tiles;
  it.b0 = p.a.group_indptr[lo];
  it.tok0 = p.a.qo_indptr[it.b0];
  while (p.a.qo_indptr[it.b0 + 1] == it.tok0) ++it.b0;
  it.row0 = it.tile * kTileRows;
  it.rows = min(kTileRows, g.rows - it.row0);
  it.tokens = g.pages * p.a.page_len;
  const int nb = blocks_of(g.pages, p.a.page_len);
  it.ja = split * bars.chunk;
  it.jb = min(nb, it.ja + bars.chunk);
  return true;
}

// Every CTA makes the plan for itself: each group's shared pages and rows, then the
// length of a block range.  With c blocks per range the launch takes about
// ceil(items / CTAs) * (c + 1.5) block times (an item's start and end cost about one
// and a half blocks); lane k tries ranges of ceil(longest / (k + 1)) blocks.
__device__ void make_plan(const PrefixParams& p, Bars& bars, GroupPlan* plan) {
  const SharedAttnParams& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int g = warp; g < a.groups; g += kThreads / 32) {
    const int pages = group_shared_pages(a, g);
    const int rows = (a.qo_indptr[a.group_indptr[g + 1]] - a.qo_indptr[a.group_indptr[g]]) * a.g;
    if (lane == 0) plan[g] = GroupPlan{rows > 0 ? pages : 0, rows, 0, 0};
  }
  __syncthreads();
  if (warp == 2) {
    int longest = 0;
    for (int g = lane; g < a.groups; g += 32) longest = max(longest, blocks_of(plan[g].pages, a.page_len));
    longest = __reduce_max_sync(0xffffffffu, longest);
    uint32_t best = 0xffffffffu;
    int chunk = 1;
    for (int k = lane + 1; k <= min(kMaxSplits, max(longest, 1)); k += 32) {
      const int c = max(1, (longest + k - 1) / k);
      long long items = 0;
      for (int g = 0; g < a.groups; ++g) {
        const int nb = blocks_of(plan[g].pages, a.page_len);
        items += (long long)((plan[g].rows + kTileRows - 1) / kTileRows) * a.Hkv * ((nb + c - 1) / c);
      }
      if (items > p.max_items && k > 1) continue;
      const long long waves = (items + gridDim.x - 1) / gridDim.x;
      const uint32_t cost = (uint32_t)min(waves * (2 * c + 3), 0xfffffffell);
      if (cost < best) {
        best = cost;
        chunk = c;
      }
    }
    const uint32_t win = __reduce_min_sync(0xffffffffu, best);
    // equal costs: the longer ranges (fewer parts)
    chunk = __reduce_max_sync(0xffffffffu, best == win ? chunk : 0);
    int run = 0;
    for (int g0 = 0; g0 < a.groups; g0 += 32) {
      const int g = g0 + lane;
      int n = 0;
      if (g < a.groups) {
        const int splits = (blocks_of(plan[g].pages, a.page_len) + chunk - 1) / chunk;
        n = (plan[g].rows + kTileRows - 1) / kTileRows * a.Hkv * splits;
        plan[g].splits = splits;
      }
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (g < a.groups) {
        plan[g].first = run + incl - n;
        if (blockIdx.x == 0) p.plan[g] = plan[g];
      }
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      bars.chunk = chunk;
      bars.total = min(run, p.max_items);
    }
  }
  __syncthreads();
}

// Ring positions of block i's K and V among n blocks, in load order.  Two row tiles use
// every block at once: K0 V0 K1 V1 ..; two block streams start with both streams' keys:
// K0 K1 V0 K2 V1 K3 ..
__device__ __forceinline__ int ring_k(bool two, int i) { return two ? 2 * i : i < 2 ? i : 2 * i - 1; }
__device__ __forceinline__ int ring_v(bool two, int i, int n) { return two ? 2 * i + 1 : i < n - 1 ? 2 * i + 2 : 2 * n - 1; }

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
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.s_full[t], 1);
      mbar_init(&bars.p_full[t], 4);
    }
    for (int s = 0; s < S::kSlots; ++s) {
      mbar_init(&bars.full[s], 1);
      mbar_init(&bars.empty[s], 1);
    }
    mbar_init(&bars.q_ready, 8);
    mbar_init(&bars.o_full, 1);
    mbar_init(&bars.drain, 1);
    bars.abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&kv_map);
  }
  if (warp == 1) {
    tmem_alloc(&bars.tmem, 512);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();                                        // the second kernel's own part needs nothing from this one
  make_plan(p, bars, plan);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    // lane = half * 8 + run: one 16-token run of one 64-column half
    const int run = lane & 7, half = lane >> 3;
    bool ok = true;
    int pushed = 0;                                     // copies into the ring so far
    Item it;
    for (int i = blockIdx.x; ok && find_item(p, bars, plan, i, it); i += gridDim.x) {
      const bool two = it.rows > 128;
      const int n = it.jb - it.ja, table = a.page_indptr[it.b0];
      for (int x = 0; ok && x < 2 * n; ++x) {
        // the x-th load: K or V of block j
        bool is_v;
        int j;
        if (two) {
          is_v = x & 1;
          j = x >> 1;
        } else if (x < min(2, n)) {
          is_v = false;
          j = x;
        } else {
          // V0 K2 V1 K3 .. ; the last two are V
          is_v = x == 2 * n - 1 || !(x & 1);
          j = x == 2 * n - 1 ? n - 1 : is_v ? (x - 2) / 2 : (x + 1) / 2;
        }
        const int tok = (it.ja + j) * kBlock + run * kRun;
        int page = a.max_pages, at = 0;                 // past the pool: zero fill
        if (tok < it.tokens) {
          const int ph = __ldg(a.page_indices + table + tok / a.page_len);
          if (ph >= 0 && ph < a.max_pages) page = ph;
          at = tok % a.page_len;
        }
        const int s = pushed % S::kSlots;
        ok = __all_sync(0xffffffffu,
                        mbar_wait_lazy(&bars.empty[s], ((pushed / S::kSlots) + 1) & 1, 100, p.wait_limit) &&
                            !gave_up(bars));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&bars.full[s], S::kSlotBytes);
        __syncwarp();
        if (half < S::kHalves)
          tma_load_4d(smem + S::kOffRing + s * S::kSlotBytes + half * S::kHalfBytes + run * (kRun * 128), &kv_map,
                      &bars.full[s], half * 64, it.h, at, 2 * page + (is_v ? 1 : 0));
        __syncwarp();
        ++pushed;
      }
    }
    if (!ok && lane == 0) give_up(bars, p, 51);
    // the copies in flight must land before the CTA can exit
    for (int x = max(0, pushed - S::kSlots); x < pushed; ++x) mbar_wait(&bars.full[x % S::kSlots], (x / S::kSlots) & 1);
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t id_qk = idesc_bf16_f32(128, kBlock, 0, 0);
    const uint32_t id_pv = idesc_bf16_f32(128, D, 0, 1);
    const uint64_t q0 = smem_desc(smem_u32(smem + S::kOffQ), 16, 1024, kSwizzle128B);
    const uint64_t k0 = smem_desc(smem_u32(smem + S::kOffRing), 16, 1024, kSwizzle128B);
    const uint64_t v0 = smem_desc(smem_u32(smem + S::kOffRing), S::kHalfBytes, 1024, kSwizzle128B);
    const bool leader = elect_one();
    bool ok = true, issued = false;
    int base = 0, items = 0;                            // ring positions before this item; items done
    int steps[2] = {0, 0};                              // phases of p_full
    auto wait_all = [&](bool x, int code) {
      ok = __all_sync(0xffffffffu, x && !gave_up(bars));
      if (!ok && lane == 0) give_up(bars, p, code);
      tc_fence_after();
      return ok;
    };
    Item it;
    for (int i = blockIdx.x; ok && find_item(p, bars, plan, i, it); i += gridDim.x) {
      const bool two = it.rows > 128;
      const int n = it.jb - it.ja;
      auto wait_slot = [&](int pos, int code) {
        return wait_all(mbar_wait(&bars.full[pos % S::kSlots], (pos / S::kSlots) & 1, p.wait_limit), code);
      };
      auto issue_s = [&](int t, int pos, bool last_use) {
        const int slot = pos % S::kSlots;
        if (leader) {
          const uint64_t qd = q0 + (uint64_t)((two ? t * S::kSlotBytes : 0u) >> 4);
          const uint64_t kd = k0 + (uint64_t)((slot * S::kSlotBytes) >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t off = (uint64_t)(((k / 4) * S::kHalfBytes + (k % 4) * 32) >> 4);
            mma_bf16_ss(tmem + kColS + 128 * t, qd + off, kd + off, id_qk, k > 0);
          }
          mma_commit(&bars.s_full[t]);
          if (last_use) mma_commit(&bars.empty[slot]);
        }
        __syncwarp();
      };
      wait_all(mbar_wait(&bars.q_ready, items & 1, p.wait_limit), 61);
      const int count[2] = {two ? n : (n + 1) / 2, two ? n : n / 2};
      for (int t = 0; ok && t < 2; ++t) {
        if (count[t] == 0) continue;
        const int pos = base + ring_k(two, two ? 0 : t);
        if (!wait_slot(pos, 62)) break;
        issue_s(t, pos, !two || t == 1);
        issued = true;
      }
      for (int x = 0; ok && x < count[0]; ++x) {
        for (int t = 0; ok && t < 2; ++t) {
          if (x >= count[t]) continue;
          const int blk = two ? x : 2 * x + t;
          const int pos = base + ring_v(two, blk, n), slot = pos % S::kSlots;
          if (!wait_slot(pos, 63)) break;
          if (!wait_all(mbar_wait(&bars.p_full[t], steps[t] & 1, p.wait_limit), 64)) break;
          ++steps[t];
          if (leader) {
            const uint64_t vd = v0 + (uint64_t)((slot * S::kSlotBytes) >> 4);
#pragma unroll
            for (int k = 0; k < kBlock / 16; ++k)
              mma_bf16_ts(tmem + kColO + D * t, tmem + kColS + 128 * t + 8 * k, vd + (uint64_t)((k * 2048) >> 4), id_pv,
                          (x > 0 || k > 0) ? 1u : 0u);
            if (!two || t == 1) mma_commit(&bars.empty[slot]);
          }
          __syncwarp();
          if (x + 1 < count[t]) {
            const int kpos = base + ring_k(two, two ? x + 1 : 2 * (x + 1) + t);
            if (!wait_slot(kpos, 65)) break;
            issue_s(t, kpos, !two || t == 1);
          }
        }
      }
      if (ok && leader) mma_commit(&bars.o_full);
      __syncwarp();
      base += 2 * n;
      ++items;
    }
    if (issued) {
      if (leader) mma_commit(&bars.drain);
      __syncwarp();
      mbar_wait(&bars.drain, 0);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax
    const int t = (warp - 4) >> 2, quarter = warp & 3;
    const int r_local = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tm = tmem + lane_base + kColS + 128 * t, o_tm = tmem + lane_base + kColO + D * t;
    bool ok = true;
    int steps = 0, items = 0;
    Item it;
    for (int i = blockIdx.x; ok && find_item(p, bars, plan, i, it); i += gridDim.x, ++items) {
      const bool two = it.rows > 128;
      const int n = it.jb - it.ja, count = two ? n : (n + 1 - t) / 2;
      const int my0 = two ? 128 * t : 0;                // this stream's first row of the tile
      if (two || t == 0) {
        // the warp's 32 query rows into the swizzled A operand, two (D = 128) or four
        // rows per load instruction; the previous item's products have all completed
        constexpr int kChunks = D / 8, kPer = 32 / kChunks;
        const int chunk = lane % kChunks;
        const uint32_t qb = smem_u32(smem + S::kOffQ + (two ? t : 0) * S::kSlotBytes) + (chunk / 8) * S::kHalfBytes;
        uint4 v[32 / kPer];
#pragma unroll
        for (int k = 0; k < 32 / kPer; ++k) {
          const int r = quarter * 32 + k * kPer + lane / kChunks, R = it.row0 + my0 + r;
          v[k] = my0 + r < it.rows
                     ? __ldg((const uint4*)((const uint16_t*)a.q +
                                            ((int64_t)(it.tok0 + R / a.g) * a.Hq + it.h * a.g + R % a.g) * D) +
                             chunk)
                     : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 32 / kPer; ++k) {
          const int r = quarter * 32 + k * kPer + lane / kChunks;
          st_shared_v4(qb + (uint32_t)r * 128u + (uint32_t)(((chunk & 7) ^ (r & 7)) << 4), v[k].x, v[k].y, v[k].z,
                       v[k].w);
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.q_ready);
      float m = -INFINITY, l = 0.0f;
      for (int x = 0; x < count; ++x) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.s_full[t], steps & 1, p.wait_limit) && !gave_up(bars));
        if (!ok) break;
        tc_fence_after();
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
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            float y0, y1;
            f2_split(ffma2(f2(__uint_as_float(s[half][c]), __uint_as_float(s[half][c + 1])), sc2, nm2), y0,
                     y1);
            y0 = fast_exp2(y0);
            y1 = fast_exp2(y1);
            if (c & 2) l1 = fadd2(l1, f2(y0, y1));
            else l0 = fadd2(l0, f2(y0, y1));
            pk[c / 2] = pack_bf16x2(y0, y1);
          }
          tmem_st32(s_tm + 32 * half, pk);
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
        if (lane == 0) mbar_arrive(&bars.p_full[t]);
        ++steps;
      }
      if (!ok) {
        if (lane == 0) give_up(bars, p, 71);
        break;
      }
      // the part: O as [column quad][row] so that a warp stores 512 contiguous bytes
      ok = __all_sync(0xffffffffu, mbar_wait(&bars.o_full, items & 1, p.wait_limit) && !gave_up(bars));
      if (!ok) {
        if (lane == 0) give_up(bars, p, 72);
        break;
      }
      tc_fence_after();
      float* part = p.parts + (int64_t)i * S::kPartFloats + t * (S::kPartFloats / 2);
      const bool valid = my0 + r_local < it.rows;
      if (count > 0) {
#pragma unroll
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
      }
      if (valid) {
        part[128 * D + r_local] = m;
        part[128 * D + 128 + r_local] = l;
      }
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
constexpr int kOwnTile = 64;              // tokens staged at a time
constexpr int kOwnStages = 2;

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

// Rows row0 .. row0 + n - 1 of request b and KV head h: joins their own parts (`parts`
// of them: O at own_o + part * part_stride + row * D, m and l at own_ml + part *
// ml_stride + row, rows counted from row0) with the shared parts, and writes the
// output.  A warp takes four rows and eight column quads at a time: both the parts
// ([quad][row]) and the output are then touched in 64-byte pieces.
template <int D>
__device__ void join_rows(const PrefixParams& p, int b, int h, int gi, int row0, int n, const float* own_o,
                          int64_t part_stride, int64_t o_row_stride, const float2* own_ml, int64_t ml_stride,
                          int64_t ml_row_stride, int parts) {
  const SharedAttnParams& a = p.a;
  const GroupPlan g = p.plan[gi];
  const int tok0 = a.qo_indptr[b];
  const int in_group = (tok0 - a.qo_indptr[a.group_indptr[gi]]) * a.g + row0;
  const int tiles = (g.rows + kTileRows - 1) / kTileRows;
  constexpr int kPart = Shape<D>::kPartFloats, kHalf = kPart / 2;
  const int groups4 = (n + 3) / 4;
  for (int idx = threadIdx.x; idx < groups4 * D; idx += kOwnThreads) {
    const int lo = idx & 31, hi = idx >> 5;
    const int r = (hi / (D / 32)) * 4 + (lo & 3), quad = (hi % (D / 32)) * 8 + (lo >> 2);
    if (r >= n) continue;
    const int rg = in_group + r, tile = rg / kTileRows, in = rg % kTileRows;
    const bool two = g.rows - tile * kTileRows > 128;
    const int t0 = two ? in >> 7 : 0, streams = two ? 1 : 2;
    const float* base = p.parts + ((int64_t)g.first + ((int64_t)h * tiles + tile) * g.splits) * kPart + t0 * kHalf;
    const int row = in & 127, shared = g.splits * streams;
    auto at = [&](int k) { return base + (two ? (int64_t)k * kPart : (int64_t)k * kHalf); };
    float M = -INFINITY;
#pragma unroll 8
    for (int k = 0; k < shared; ++k) M = fmaxf(M, __ldcg(at(k) + 128 * D + row));
    for (int k = 0; k < parts; ++k) M = fmaxf(M, own_ml[k * ml_stride + r * ml_row_stride].x);
    const float base_m = M == -INFINITY ? 0.0f : M;
    float L = 0.0f, o0 = 0.0f, o1 = 0.0f, o2 = 0.0f, o3 = 0.0f;
    auto add = [&](float m, float l, const float4 v) {
      const float w = fast_exp2(m - base_m);
      L = fmaf(w, l, L);
      o0 = fmaf(w, v.x, o0);
      o1 = fmaf(w, v.y, o1);
      o2 = fmaf(w, v.z, o2);
      o3 = fmaf(w, v.w, o3);
    };
#pragma unroll 4
    for (int k = 0; k < shared; ++k) {
      const float* s = at(k);
      const float m = __ldcg(s + 128 * D + row), l = __ldcg(s + 128 * D + 128 + row);
      if (m != -INFINITY) add(m, l, __ldcg((const float4*)s + quad * 128 + row));
    }
    for (int k = 0; k < parts; ++k) {
      const float2 ml = own_ml[k * ml_stride + r * ml_row_stride];
      if (ml.x != -INFINITY) add(ml.x, ml.y, *(const float4*)(own_o + k * part_stride + r * o_row_stride + quad * 4));
    }
    const float inv = L > 0.0f ? 1.0f / L : L == L ? 0.0f : L;   // nothing seen: 0
    const int R = row0 + r;
    *(uint2*)((uint16_t*)a.out + ((int64_t)(tok0 + R / a.g) * a.Hq + h * a.g + R % a.g) * D + quad * 4) =
        make_uint2(pack_bf16x2(o0 * inv, o1 * inv), pack_bf16x2(o2 * inv, o3 * inv));
  }
}

// WR of the four warps split the CTA's 16 WR rows, the others the staged tokens.
template <int D, int WR>
__global__ void __launch_bounds__(kOwnThreads) own_attn_kernel(const PrefixParams p) {
  constexpr int WT = 4 / WR, kRows = 16 * WR, kChunks = D / 8, kRowBytes = D * 2;
  constexpr uint32_t kTileBytes = kOwnTile * kRowBytes;         // K or V
  extern __shared__ __align__(16) uint8_t stage[];
  __shared__ float2 ml[WT][kRows];
  const SharedAttnParams& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  const int wr = warp % WR, wt = warp / WR;
  const int b = blockIdx.x / p.request_tiles, row0 = blockIdx.x % p.request_tiles * kRows, h = blockIdx.y;
  const int tok0 = a.qo_indptr[b], n_tok = a.qo_indptr[b + 1] - tok0, total_rows = n_tok * a.g;
  pdl_trigger();
  if (row0 >= total_rows) {
    pdl_wait();                                         // no CTA ends before the first kernel has: what follows may
    return;                                             // wait for this one alone
  }
  const int rows = min(kRows, total_rows - row0);
  const int gi = group_of(a, b);
  const int shared = group_shared_pages(a, gi);
  const int table = a.page_indptr[b] + shared;
  const int len = max(0, kv_tokens(a, b) - shared * a.page_len), prefix = len - n_tok;
  const int n_tiles = (len + kOwnTile - 1) / kOwnTile;
  const int j0 = (int)((int64_t)n_tiles * blockIdx.z / p.own_splits);
  const int j1 = (int)((int64_t)n_tiles * (blockIdx.z + 1) / p.own_splits);
  const uint32_t smem0 = smem_u32(stage);
  const int64_t tok_elems = (int64_t)a.Hkv * D;
  const uint16_t* kv = (const uint16_t*)a.kv + (int64_t)h * D;

  auto load_tile = [&](int j) {
    const uint32_t buf = smem0 + (j % kOwnStages) * 2 * kTileBytes;
#pragma unroll
    for (int e0 = 0; e0 < kOwnTile * kChunks; e0 += kOwnThreads) {
      const int e = e0 + threadIdx.x, t = e / kChunks, c = e % kChunks, tok = j * kOwnTile + t;
      const uint16_t* src = kv;
      bool valid = tok < len;
      if (valid) {
        const int page = __ldg(a.page_indices + table + tok / a.page_len);
        valid = page >= 0 && page < a.max_pages;
        if (valid) src = kv + ((int64_t)page * 2 * a.page_len + tok % a.page_len) * tok_elems + c * 8;
      }
      const uint32_t dst = buf + t * kRowBytes + ((c ^ (t & 7)) << 4);
      cp_async16(dst, src, valid);
      cp_async16(dst + kTileBytes, valid ? src + a.page_len * tok_elems : src, valid);
    }
    cp_async_commit();
  };

  for (int s = 0; s < kOwnStages - 1; ++s) {
    if (j0 + s < j1) load_tile(j0 + s);
    else cp_async_commit();
  }
  // the warp's 16 query rows as A fragments; rows past the request's are zero
  uint32_t qa[D / 16][4];
  int node[2];
  const uint64_t* mask[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = wr * 16 + gq + 8 * i, R = row0 + r;
    const bool valid = r < rows;
    node[i] = valid ? R / a.g : 0;
    mask[i] = a.mask_bits ? a.mask_bits + (int64_t)(tok0 + node[i]) * a.mask_words : nullptr;
    const uint16_t* q = (const uint16_t*)a.q + ((int64_t)(tok0 + node[i]) * a.Hq + h * a.g + (valid ? R % a.g : 0)) * D;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qa[k][i] = valid ? __ldg((const uint32_t*)(q + 16 * k + 2 * tq)) : 0u;
      qa[k][2 + i] = valid ? __ldg((const uint32_t*)(q + 16 * k + 8 + 2 * tq)) : 0u;
    }
  }
  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  const int mi = lane >> 3, rr = lane & 7;

  for (int j = j0; j < j1; ++j) {
    if (j + kOwnStages - 1 < j1) load_tile(j + kOwnStages - 1);
    else cp_async_commit();
    cp_async_wait<kOwnStages - 1>();
    __syncthreads();
    const uint32_t kb = smem0 + (j % kOwnStages) * 2 * kTileBytes, vb = kb + kTileBytes;
    const int c0 = j * kOwnTile, t0 = wt * (kOwnTile / WT);
    float s[WR][2][4];
#pragma unroll
    for (int c = 0; c < WR; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c][e >> 2][e & 3] = 0.0f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int c = 0; c < WR; ++c) {
        const int t = t0 + 16 * c + rr + 8 * (mi >> 1);
        uint32_t r0, r1, r2, r3;
        ldmatrix_x4(kb + t * kRowBytes + (((2 * k + (mi & 1)) ^ (t & 7)) << 4), r0, r1, r2, r3);
        mma_m16n8k16(s[c][0], qa[k], r0, r1);
        mma_m16n8k16(s[c][1], qa[k], r2, r3);
      }
    const bool masked = c0 + kOwnTile > prefix;         // tree slots or the end in this tile
    uint64_t seen[2] = {~0ull, ~0ull};
    if (masked) {
#pragma unroll
      for (int i = 0; i < 2; ++i) seen[i] = seen_columns(a, mask[i], node[i], c0, prefix, len);
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < WR; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float& x = s[c][e >> 2][e & 3];
        const int i = (e >> 1) & 1, col = t0 + 16 * c + 8 * (e >> 2) + 2 * tq + (e & 1);
        x = (seen[i] >> col) & 1ull ? x * p.scale_log2 : -INFINITY;
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
    for (int i = 0; i < D / 8; ++i) {
      o[i][0] *= keep[0];
      o[i][1] *= keep[0];
      o[i][2] *= keep[1];
      o[i][3] *= keep[1];
    }
#pragma unroll
    for (int c = 0; c < WR; ++c)
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
      for (int c = 0; c < WR; ++c) {
        const uint32_t pa[4] = {pack_bf16x2(s[c][0][0], s[c][0][1]), pack_bf16x2(s[c][0][2], s[c][0][3]),
                                pack_bf16x2(s[c][1][0], s[c][1][1]), pack_bf16x2(s[c][1][2], s[c][1][3])};
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          const int t = t0 + 16 * c + rr + 8 * (mi & 1);
          uint32_t r0, r1, r2, r3;
          ldmatrix_x4_trans(vb + t * kRowBytes + (((2 * d + (mi >> 1)) ^ (t & 7)) << 4), r0, r1, r2, r3);
          mma_m16n8k16(o[2 * d], pa, r0, r1);
          mma_m16n8k16(o[2 * d + 1], pa, r2, r3);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < WR; ++c)
#pragma unroll
        for (int u = 0; u < 16; ++u) {                  // token u of the 16: its lane of the quad, its element
          const float p0 = __shfl_sync(0xffffffffu, s[c][u >> 3][u & 1], (lane & ~3) | ((u & 7) >> 1));
          const float p1 = __shfl_sync(0xffffffffu, s[c][u >> 3][2 + (u & 1)], (lane & ~3) | ((u & 7) >> 1));
          const int t = t0 + 16 * c + u;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            uint32_t w;
            asm volatile("ld.shared.b32 %0, [%1];"
                         : "=r"(w)
                         : "r"(vb + t * kRowBytes + ((d ^ (t & 7)) << 4) + 4 * tq));
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
    if (tq == 0) ml[wt][r] = make_float2(m[i], l[i]);
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
      *(float2*)(os + (wt * kRows + r) * D + 8 * d + 2 * tq) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
  }
  __syncthreads();
  if (p.own_splits > 1) {
    // a slice of the own columns: one part per row for the join kernel
    for (int e = threadIdx.x; e < rows * (D / 4); e += kOwnThreads) {
      const int r = e / (D / 4), quad = e % (D / 4), R = row0 + r;
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
      const int64_t row = (int64_t)(tok0 + R / a.g) * a.Hq + h * a.g + R % a.g, part = row * p.own_splits + blockIdx.z;
      *(float4*)(p.own_o + part * D + quad * 4) = acc;
      if (quad == 0) p.own_ml[part] = make_float2(M, L);
    }
    pdl_wait();
    return;
  }
  pdl_wait();                                           // the shared parts are complete
  join_rows<D>(p, b, h, gi, row0, rows, os, kRows * D, D, &ml[0][0], kRows, 1, WT);
}

// After own_attn_kernel with several slices: joins each row's parts.
template <int D>
__global__ void __launch_bounds__(kOwnThreads) join_parts_kernel(const PrefixParams p) {
  const SharedAttnParams& a = p.a;
  pdl_trigger();
  pdl_wait();
  constexpr int kRows = 16;
  const int b = blockIdx.x / p.request_tiles, row0 = blockIdx.x % p.request_tiles * kRows, h = blockIdx.y;
  const int tok0 = a.qo_indptr[b], total_rows = (a.qo_indptr[b + 1] - tok0) * a.g;
  if (row0 >= total_rows) return;
  // a request's row R is row (tok0 + R / g) * Hq + h * g + R % g of the parts: uniform
  // strides within one token's heads only, so take the token's heads one by one
  const int n = min(kRows, total_rows - row0);
  for (int r = 0; r < n;) {
    const int R = row0 + r, k = min(n - r, a.g - R % a.g);
    const int64_t row = (int64_t)(tok0 + R / a.g) * a.Hq + h * a.g + R % a.g;
    join_rows<D>(p, b, h, group_of(a, b), R, k, p.own_o + row * p.own_splits * D, D, (int64_t)p.own_splits * D,
                 p.own_ml + row * p.own_splits, 1, p.own_splits, p.own_splits);
    r += k;
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
  // own columns: about three CTAs per SM, each with two tiles at least
  const int64_t ctas = (int64_t)batch * f.request_tiles * Hkv;
  const int own = max_own_len > 0 ? max_own_len : max_kv_len;
  f.own_splits = (int)std::max<int64_t>(
      1, std::min<int64_t>({3ll * f.ctas / std::max<int64_t>(ctas, 1), (own + 2 * kOwnTile - 1) / (2 * kOwnTile), 32}));
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
  constexpr size_t smem = (size_t)kOwnStages * 2 * kOwnTile * D * 2;
  static_assert(smem >= (size_t)64 * D * 4, "the stages hold the warps' O");
  if (int rc = ensure_smem_attr((const void*)own_attn_kernel<D, WR>, smem)) return rc;
  PTS_CUDA_TRY(launch_pdl(own_attn_kernel<D, WR>, dim3(p.a.batch * p.request_tiles, p.a.Hkv, p.own_splits),
                          dim3(kOwnThreads), smem, stream, p));
  return launch_status("own_attn_kernel");
}

template <int D>
int launch_prefix(PrefixParams p, const PrefixPlan& f, int max_qo_len, cudaStream_t stream) {
  const SharedAttnParams& a = p.a;
  CUtensorMap map;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)a.Hkv, (cuuint64_t)a.page_len, (cuuint64_t)a.max_pages * 2};
  const cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)a.Hkv * D * 2, (cuuint64_t)a.page_len * a.Hkv * D * 2};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)kRun, 1};
  if (int rc = encode_tiled_bf16_sw128(&map, 4, a.kv, dims, strides, box)) return rc;
  if (int rc = ensure_smem_attr((const void*)prefix_attn_kernel<D>, Shape<D>::kSmem)) return rc;
  PTS_CUDA_TRY(launch_pdl(prefix_attn_kernel<D>, dim3(f.ctas), dim3(kThreads), Shape<D>::kSmem, stream, p, map));
  if (int rc = launch_status("prefix_attn_kernel")) return rc;
  int rc = f.own_rows == 16 ? launch_own<D, 1>(p, stream) : f.own_rows == 32 ? launch_own<D, 2>(p, stream)
                                                                            : launch_own<D, 4>(p, stream);
  if (rc || p.own_splits == 1) return rc;
  PrefixParams j = p;
  j.request_tiles = (int)(((int64_t)max_qo_len * a.g + 15) / 16);
  PTS_CUDA_TRY(launch_pdl(join_parts_kernel<D>, dim3(a.batch * j.request_tiles, a.Hkv), dim3(kOwnThreads), 0, stream, j));
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
  char* ws = (char*)workspace;
  PrefixParams p{};
  p.a = a;
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
  return a.D == 128 ? launch_prefix<128>(p, f, max_qo_len, stream) : launch_prefix<64>(p, f, max_qo_len, stream);
}

}  // namespace pts
