// Tree attention for requests that share leading pages, any supported type and
// shape (fp32 or bf16, head_dim a multiple of 32 up to 256, any page length): the
// fp32 path of the small configurations, and the entry point.
//
// parts_kernel: a CTA holds 32 query rows (8 per warp) and one slice of a column
// set -- the shared columns of the rows' group, or one request's own -- and walks
// it in tiles of 32 tokens staged in shared memory as fp32.  A lane owns one token
// of the tile for the scores (8 rows at a time, so each K value read serves 8
// products) and D/32 output dimensions for the sums.  Row max, row sum and O stay in
// registers and go to the workspace as one part; join_kernel joins a row's parts.
// Bound by shared-memory reads (9 16-byte reads per 32 products of four) and, at the
// small sizes it is for, by latency: 8 requests of 15 nodes, 128 shared and 40 own tokens,
// 2 KV heads of 64 in fp32 take 19 us with the join.
#include "attn_shared.cuh"

#include <algorithm>

namespace pts {
namespace {

constexpr int kWarps = 4;
constexpr int kWarpRows = 8;
constexpr int kRows = kWarps * kWarpRows;
constexpr int kTile = 32;                // tokens per tile

struct PartsParams {
  SharedAttnParams a;
  int splits;              // slices of a column set
  int group_tiles;         // CTAs in x for the groups' rows; the rest are the requests'
  int request_tiles;       // CTAs per request
  float* part_o;           // [T * Hq][2 * splits][D]
  float2* part_ml;         // [T * Hq][2 * splits]
};

template <class T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) {
  return *reinterpret_cast<const float4*>(p);
}
template <>
__device__ __forceinline__ float4 load4<uint16_t>(const uint16_t* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(bf16_bits_to_float(v.x & 0xffffu), bf16_bits_to_float(v.x >> 16),
                     bf16_bits_to_float(v.y & 0xffffu), bf16_bits_to_float(v.y >> 16));
}
__device__ __forceinline__ void store_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_value(uint16_t* p, float v) { *p = float_to_bf16_bits(v); }

// Shared memory: K and V rows of D + 4 floats (the pad spreads a column over the
// banks), Q rows of D, P [row][token].
template <int PER>
constexpr int smem_floats() {
  return 2 * kTile * (PER * 32 + 4) + kRows * PER * 32 + kRows * kTile;
}

template <class T, int PER>
__global__ void __launch_bounds__(kWarps * 32) parts_kernel(const PartsParams p) {
  constexpr int D = PER * 32, kStride = D + 4;
  extern __shared__ float smem[];
  float* ks = smem;
  float* vs = ks + kTile * kStride;
  float* qs = vs + kTile * kStride;
  float* ps = qs + kRows * D;
  const SharedAttnParams& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, split = blockIdx.z;
  // the rows: a tile of a group's tokens x heads, or of one request's
  int tok0, n_tok, row0, b0, first_page, c0, c1, prefix, kv_len;
  bool own;
  if ((int)blockIdx.x < p.group_tiles) {
    own = false;
    int left = blockIdx.x, gi = 0;
    for (; gi < a.groups; ++gi) {
      const int2 range = group_requests(a, gi);
      n_tok = a.qo_indptr[range.y] - a.qo_indptr[range.x];
      const int tiles = (n_tok * a.g + kRows - 1) / kRows;
      if (left < tiles) break;
      left -= tiles;
    }
    if (gi == a.groups) return;
    b0 = group_requests(a, gi).x;
    tok0 = a.qo_indptr[b0];
    row0 = left * kRows;
    // the table of the group's first request with rows
    while (a.qo_indptr[b0 + 1] == tok0) ++b0;
    first_page = a.page_indptr[b0];
    kv_len = group_shared_pages(a, gi) * a.page_len;
    prefix = kv_len;
  } else {
    own = true;
    const int u = blockIdx.x - p.group_tiles;
    b0 = u / p.request_tiles;
    row0 = (u % p.request_tiles) * kRows;
    tok0 = a.qo_indptr[b0];
    n_tok = a.qo_indptr[b0 + 1] - tok0;
    if (row0 >= n_tok * a.g) return;
    const int shared = group_shared_pages(a, group_of(a, b0));
    first_page = a.page_indptr[b0] + shared;
    kv_len = kv_tokens(a, b0) - shared * a.page_len;    // tokens after the shared pages
    prefix = kv_len - n_tok;
  }
  {
    const int tiles = (max(kv_len, 0) + kTile - 1) / kTile;
    c0 = (int)((int64_t)tiles * split / p.splits) * kTile;
    c1 = min((int)((int64_t)tiles * (split + 1) / p.splits) * kTile, kv_len);
  }
  const int rows = min(kRows, n_tok * a.g - row0);
  const T* q = (const T*)a.q;
  for (int e = threadIdx.x; e < kRows * (D / 4); e += kWarps * 32) {
    const int r = e / (D / 4), d = e % (D / 4) * 4;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < rows) {
      const int R = row0 + r;
      v = load4(q + ((int64_t)(tok0 + R / a.g) * a.Hq + h * a.g + R % a.g) * D + d);
    }
    *reinterpret_cast<float4*>(qs + r * D + d) = v;
  }
  float m[kWarpRows], l[kWarpRows], o[kWarpRows][PER];
#pragma unroll
  for (int r = 0; r < kWarpRows; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[r][i] = 0.0f;
  }
  const int64_t tok_elems = (int64_t)a.Hkv * D;
  for (int c = c0; c < c1; c += kTile) {
    bool odd = false;                                   // a value that 0 * v does not cancel
    __syncthreads();
#pragma unroll 4
    for (int e = threadIdx.x; e < kTile * (D / 4); e += kWarps * 32) {
      const int t = e / (D / 4), d = e % (D / 4) * 4;
      float4 kx = make_float4(0.0f, 0.0f, 0.0f, 0.0f), vx = kx;
      if (c + t < c1) {                                 // slots past the end are not read
        const int page = a.page_indices[first_page + (c + t) / a.page_len];
        if (page >= 0 && page < a.max_pages) {
          const T* k = (const T*)a.kv + ((int64_t)page * 2 * a.page_len + (c + t) % a.page_len) * tok_elems +
                       (int64_t)h * D + d;
          kx = load4(k);
          vx = load4(k + (int64_t)a.page_len * tok_elems);
        }
      }
      *reinterpret_cast<float4*>(ks + t * kStride + d) = kx;
      *reinterpret_cast<float4*>(vs + t * kStride + d) = vx;
      odd |= !(fabsf(vx.x) < INFINITY && fabsf(vx.y) < INFINITY && fabsf(vx.z) < INFINITY && fabsf(vx.w) < INFINITY);
    }
    odd = __syncthreads_or(odd) && own;                 // the shared columns have no mask
    float s[kWarpRows];
#pragma unroll
    for (int r = 0; r < kWarpRows; ++r) s[r] = 0.0f;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      const float4 k = *reinterpret_cast<const float4*>(ks + lane * kStride + d);
#pragma unroll
      for (int r = 0; r < kWarpRows; ++r) {
        const float4 x = *reinterpret_cast<const float4*>(qs + (warp * kWarpRows + r) * D + d);
        s[r] = fmaf(x.x, k.x, s[r]);
        s[r] = fmaf(x.y, k.y, s[r]);
        s[r] = fmaf(x.z, k.z, s[r]);
        s[r] = fmaf(x.w, k.w, s[r]);
      }
    }
    const int j = c + lane;
#pragma unroll
    for (int r = 0; r < kWarpRows; ++r) {
      bool seen = j < c1;
      if (own && seen && j >= prefix) {
        const int node = (row0 + warp * kWarpRows + r) / a.g, t = j - prefix;
        if (node >= n_tok) seen = false;
        else if (!a.mask_bits) seen = t <= node;
        else
          seen = (t >> 6) < a.mask_words &&
                 ((a.mask_bits[(int64_t)(tok0 + node) * a.mask_words + (t >> 6)] >> (t & 63)) & 1ull);
      }
      const float x = seen ? s[r] * a.scale : -INFINITY;
      float top = x;
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float nm = fmaxf(m[r], top);
      const float base = nm == -INFINITY ? 0.0f : nm;   // a row that has seen nothing yet
      const float e = expf(x - base);
      const float keep = expf(m[r] - base);
      float sum = e;
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      l[r] = l[r] * keep + sum;
      m[r] = nm;
#pragma unroll
      for (int i = 0; i < PER; ++i) o[r][i] *= keep;
      ps[(warp * kWarpRows + r) * kTile + lane] = e;
    }
    __syncwarp();
    if (odd) {
      // infinities or NaN among the values: a masked slot's must not reach the row
      for (int t = 0; t < kTile; ++t)
#pragma unroll
        for (int r = 0; r < kWarpRows; ++r) {
          const float e = ps[(warp * kWarpRows + r) * kTile + t];
          if (e == 0.0f) continue;
#pragma unroll
          for (int i = 0; i < PER; ++i) o[r][i] = fmaf(e, vs[t * kStride + lane + 32 * i], o[r][i]);
        }
      __syncwarp();
      continue;
    }
#pragma unroll 2
    for (int t = 0; t < kTile; t += 4) {
      float v[4][PER];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < PER; ++i) v[u][i] = vs[(t + u) * kStride + lane + 32 * i];
#pragma unroll
      for (int r = 0; r < kWarpRows; ++r) {
        const float4 e = *reinterpret_cast<const float4*>(ps + (warp * kWarpRows + r) * kTile + t);
#pragma unroll
        for (int i = 0; i < PER; ++i)
          o[r][i] = fmaf(e.w, v[3][i], fmaf(e.z, v[2][i], fmaf(e.y, v[1][i], fmaf(e.x, v[0][i], o[r][i]))));
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int r = 0; r < kWarpRows; ++r) {
    const int R = row0 + warp * kWarpRows + r;
    if (R >= n_tok * a.g) continue;
    const int64_t row = (int64_t)(tok0 + R / a.g) * a.Hq + h * a.g + R % a.g;
    const int64_t slot = row * 2 * p.splits + (own ? p.splits : 0) + split;
    if (lane == 0) p.part_ml[slot] = make_float2(m[r], l[r]);
    if (m[r] == -INFINITY) continue;                    // an empty part has no O
#pragma unroll
    for (int i = 0; i < PER; ++i) p.part_o[slot * D + lane + 32 * i] = o[r][i];
  }
}

// One warp per row: its parts in slice order, shared columns first.
template <class T>
__global__ void __launch_bounds__(256) join_kernel(const PartsParams p) {
  const SharedAttnParams& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (int64_t)a.qo_indptr[a.batch] * a.Hq) return;
  const int n = 2 * p.splits;
  const float2* ml = p.part_ml + row * n;
  float M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, ml[i].x);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
  T* out = (T*)a.out + row * a.D;
  float acc[8], L = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  for (int k = 0; k < n; ++k) {
    const float2 x = ml[k];
    if (x.x == -INFINITY && x.y == 0.0f) continue;      // (a NaN sum goes on to the row)
    const float w = expf(x.x - M);
    L += w * x.y;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.D) acc[i] = fmaf(w, p.part_o[(row * n + k) * a.D + lane + 32 * i], acc[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)                           // a row that sees nothing is 0
    if (lane + 32 * i < a.D) store_value(out + lane + 32 * i, L > 0.0f ? acc[i] / L : L == L ? 0.0f : L);
}

struct Plan {
  int splits, group_tiles, request_tiles;
  size_t part_o, bytes;
};

// Slices so that about four CTAs per SM run, each of a tile at least: at the small sizes
// this kernel is for, a tile's latency is what counts (8 requests of 15 nodes with 128 shared
// tokens: 34 us in one slice of the columns, 17 in six).
Plan make_plan(int batch, int groups, int total_q, int max_qo_len, int max_kv_len, int Hq, int Hkv, int D) {
  Plan pl;
  const int g = Hq / Hkv;
  pl.group_tiles = (int)(((int64_t)total_q * g + kRows - 1) / kRows) + groups;
  pl.request_tiles = (int)(((int64_t)max_qo_len * g + kRows - 1) / kRows);
  const int64_t ctas = ((int64_t)pl.group_tiles + (int64_t)batch * pl.request_tiles) * Hkv;
  const int64_t most = std::max<int64_t>(1, ((int64_t)max_kv_len + kTile - 1) / kTile);
  pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>({4 * 148 / std::max<int64_t>(ctas, 1), most, 32}));
  const size_t slots = (size_t)total_q * Hq * 2 * pl.splits;
  pl.part_o = align_up(slots * sizeof(float2), 256);
  pl.bytes = pl.part_o + slots * D * sizeof(float);
  return pl;
}

template <class T, int PER>
int launch_parts(const PartsParams& p, dim3 grid, cudaStream_t stream) {
  constexpr size_t smem = smem_floats<PER>() * sizeof(float);
  if (smem > 48 * 1024)
    if (int rc = ensure_smem_attr((const void*)parts_kernel<T, PER>, smem)) return rc;
  parts_kernel<T, PER><<<grid, kWarps * 32, smem, stream>>>(p);
  return launch_status("parts_kernel");
}

template <class T>
int launch_any(const PartsParams& p, dim3 grid, int total_q, cudaStream_t stream) {
  int rc = PTS_ERR_UNSUPPORTED;
  switch (p.a.D / 32) {
    case 1: rc = launch_parts<T, 1>(p, grid, stream); break;
    case 2: rc = launch_parts<T, 2>(p, grid, stream); break;
    case 3: rc = launch_parts<T, 3>(p, grid, stream); break;
    case 4: rc = launch_parts<T, 4>(p, grid, stream); break;
    case 5: rc = launch_parts<T, 5>(p, grid, stream); break;
    case 6: rc = launch_parts<T, 6>(p, grid, stream); break;
    case 7: rc = launch_parts<T, 7>(p, grid, stream); break;
    case 8: rc = launch_parts<T, 8>(p, grid, stream); break;
  }
  if (rc) return rc;
  join_kernel<T><<<(unsigned)(((int64_t)total_q * p.a.Hq + 7) / 8), 256, 0, stream>>>(p);
  return launch_status("join_kernel");
}

}  // namespace
}  // namespace pts

using namespace pts;

extern "C" size_t pts_tree_attn_shared_workspace_size(int batch, int num_groups, int total_q, int max_qo_len,
                                                      int max_kv_len, int max_own_len, int num_qo_heads,
                                                      int num_kv_heads, int head_dim, int page_len, int elem_bytes) {
  if (batch <= 0 || num_groups <= 0 || total_q <= 0 || max_qo_len <= 0 || max_kv_len <= 0 || num_qo_heads <= 0 ||
      num_kv_heads <= 0 || num_qo_heads % num_kv_heads || head_dim <= 0)
    return 0;
  max_qo_len = std::min(max_qo_len, total_q);           // (a request has at most all rows)
  if (prefix_attn_supports(head_dim, page_len, elem_bytes))
    return prefix_attn_workspace(batch, num_groups, total_q, max_qo_len, max_kv_len, max_own_len, num_qo_heads,
                                 num_kv_heads, head_dim);
  return make_plan(batch, num_groups, total_q, max_qo_len, max_kv_len, num_qo_heads, num_kv_heads, head_dim).bytes;
}

extern "C" int pts_tree_attn_run_shared(const pts_shared_attn_args* args, void* workspace, size_t workspace_bytes,
                                        pts_stream_t stream) {
  PTS_CHECK_ARG(args, "null arguments");
  const pts_shared_attn_args& x = *args;
  PTS_CHECK_ARG(x.q && x.kv_layer && x.qo_indptr && x.page_indptr && x.page_indices && x.last_page_len && x.out, "null pointer");
  PTS_CHECK_ARG(x.group_indptr && x.shared_pages && x.num_groups > 0, "groups need group_indptr and shared_pages");
  PTS_CHECK_ARG(x.batch > 0 && x.total_q > 0 && x.max_qo_len > 0 && x.max_kv_len > 0 && x.max_own_len >= 0, "bad sizes");
  PTS_CHECK_ARG(x.num_qo_heads > 0 && x.num_kv_heads > 0 && x.num_qo_heads % x.num_kv_heads == 0, "bad head counts");
  PTS_CHECK_ARG(x.page_len > 0 && x.max_pages > 0, "bad page sizes");
  if (x.head_dim <= 0 || x.head_dim % 32 || x.head_dim > 256)
    return set_error(PTS_ERR_UNSUPPORTED, "head_dim %d (a multiple of 32 up to 256)", x.head_dim);
  if (x.elem_bytes != 2 && x.elem_bytes != 4) return set_error(PTS_ERR_UNSUPPORTED, "element size %d", x.elem_bytes);
  if (x.mask_bits) {
    if (x.max_qo_len > PTS_MAX_TREE_NODES)
      return set_error(PTS_ERR_CAPACITY, "tree of %d rows above %d", x.max_qo_len, PTS_MAX_TREE_NODES);
    PTS_CHECK_ARG(x.mask_words >= (x.max_qo_len + 63) / 64, "mask_words %d too small for %d rows", x.mask_words,
                  x.max_qo_len);
  }
  PTS_CHECK_ARG((((uintptr_t)x.q | (uintptr_t)x.kv_layer | (uintptr_t)x.out) & 15) == 0,
                "q, kv_layer and out must be 16-byte aligned");
  PTS_CHECK_ARG(((uintptr_t)workspace & 255) == 0, "workspace must be 256-byte aligned");
  if (x.num_kv_heads > 65535) return set_error(PTS_ERR_CAPACITY, "grid too large");
  const size_t need = pts_tree_attn_shared_workspace_size(x.batch, x.num_groups, x.total_q, x.max_qo_len, x.max_kv_len,
                                                          x.max_own_len, x.num_qo_heads, x.num_kv_heads, x.head_dim, x.page_len,
                                                          x.elem_bytes);
  if ((!workspace && need) || workspace_bytes < need)
    return set_error(PTS_ERR_CAPACITY, "workspace of %zu bytes (%zu needed)", workspace_bytes, need);
  SharedAttnParams a{};
  a.q = x.q;
  a.kv = x.kv_layer;
  a.qo_indptr = x.qo_indptr;
  a.page_indptr = x.page_indptr;
  a.page_indices = x.page_indices;
  a.last_page_len = x.last_page_len;
  a.mask_bits = x.mask_bits;
  a.mask_words = x.mask_words;
  a.out = x.out;
  a.group_indptr = x.group_indptr;
  a.shared_pages = x.shared_pages;
  a.batch = x.batch;
  a.groups = x.num_groups;
  a.Hq = x.num_qo_heads;
  a.Hkv = x.num_kv_heads;
  a.g = x.num_qo_heads / x.num_kv_heads;
  a.D = x.head_dim;
  a.page_len = x.page_len;
  a.max_pages = x.max_pages;
  a.scale = x.sm_scale;
  const int max_qo_len = std::min(x.max_qo_len, x.total_q);
  if (prefix_attn_supports(x.head_dim, x.page_len, x.elem_bytes))
    return prefix_attn_launch(a, x.total_q, max_qo_len, x.max_kv_len, x.max_own_len, workspace, x.error, (cudaStream_t)stream);
  const Plan pl = make_plan(x.batch, x.num_groups, x.total_q, max_qo_len, x.max_kv_len, x.num_qo_heads, x.num_kv_heads, x.head_dim);
  const int64_t gx = (int64_t)pl.group_tiles + (int64_t)x.batch * pl.request_tiles;
  if (gx > 2147483647ll) return set_error(PTS_ERR_CAPACITY, "grid too large");
  PartsParams p{a, pl.splits, pl.group_tiles, pl.request_tiles, (float*)((char*)workspace + pl.part_o),
                (float2*)workspace};
  const dim3 grid((unsigned)gx, x.num_kv_heads, pl.splits);
  return x.elem_bytes == 4 ? launch_any<float>(p, grid, x.total_q, (cudaStream_t)stream)
                         : launch_any<uint16_t>(p, grid, x.total_q, (cudaStream_t)stream);
}
