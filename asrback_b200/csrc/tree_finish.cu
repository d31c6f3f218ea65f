// What comes after the draft-tree attention, sm_100a: the items whose tiles lay in
// several CTAs are merged from their parts, and (with weights) the scaled scores
// that the attention left become accumulated weights.
//
// A kernel of its own, so that the attention's CTAs end without waiting for one
// another's parts and the merges run on the whole GPU at once. It moves the parts
// once, 4 bytes per score and 8 per weight, but latency bounds it: a CTA has one
// item, finds its place in the tile list while the attention still runs, and then
// loads all it needs (references, sums and outputs of the parts, scores) at once.
// Measured, behind the attention: 3 us for 1 row x 6 nodes, 5 for 64 rows x 16
// nodes, 7.5 for 8 rows x 64 nodes (13 MB of parts) and for 64 rows x 1 node with
// weights (1536 CTAs).
#include "capi_internal.h"
#include "tree_attention.cuh"

#include <algorithm>

namespace asrback {
namespace {

using namespace tree;

constexpr int kThreads = 128;
constexpr int kMaxRows = 16;            // rows of a CTA
constexpr int kKeysPer = 4 * kThreads;  // keys of a CTA

// Shared memory of a CTA.
struct Shared {
  float part_m[kThreads], part_l[kThreads];  // [group of parts][row]
  float row_m[kMaxRows], row_l[kMaxRows];    // the rows' references and sums
  unsigned long long masks[kMaxRows];
  int tiles[2][kThreads / 32];  // warps' shares: of the rows before the CTA's, of all
};

// The item's place in the list of all items' tiles.
__device__ __forceinline__ Sharers find_place(const TreeParams& p, int b, int index, int tiles,
                                              Shared& s) {
  const int tid = threadIdx.x, per_row = p.kv_heads * p.mblocks;
  int before = 0, all = 0;
  for (int row = tid; row < p.batch; row += kThreads) {
    const RowSpan span = row_span(p, row);
    const int n = row_tiles(span.length + span.count) * per_row;
    all += n;
    before += row < b ? n : 0;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  all = __reduce_add_sync(0xffffffffu, all);
  if (tid % 32 == 0) s.tiles[0][tid / 32] = before, s.tiles[1][tid / 32] = all;
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) before += s.tiles[0][w], all += s.tiles[1][w];
  const Split split(p, all);
  return Sharers(split, before + split.lead * b * per_row + index * (tiles + split.lead), tiles);
}

// References and sums of the item's rows row0.. over its parts: a thread per row
// and group of parts.
template <int D, int kRows>
__device__ __forceinline__ void join_sums(const TreeParams& p, const Sharers& by, int row0,
                                          int rows, Shared& s) {
  constexpr int kGroups = kThreads / kRows, kDeep = 4;
  const int tid = threadIdx.x, r = tid % kRows, group = tid / kRows;
  float m = -INFINITY, l = 0.f;
  if (r < rows && by.count > 1) {
    for (int c0 = group; c0 < by.count; c0 += kGroups * kDeep) {
      float m2[kDeep], l2[kDeep];
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const int c = c0 + u * kGroups;
        const float* x = Parts<D>::of(p, by, min(c, by.count - 1)) + row0 + r;
        m2[u] = c < by.count ? x[0] : -INFINITY;
        l2[u] = c < by.count ? x[p.block_rows] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const float now = fmaxf(m, m2[u]), ref = now == -INFINITY ? 0.f : now;
        l = l * fast_exp2(m - ref) + l2[u] * fast_exp2(m2[u] - ref);
        m = now;
      }
    }
  }
  s.part_m[tid] = m;
  s.part_l[tid] = l;
  __syncthreads();
  if (tid < min(rows, kRows)) {
    m = -INFINITY;
#pragma unroll 8
    for (int g = 0; g < kGroups; ++g) m = fmaxf(m, s.part_m[g * kRows + tid]);
    const float ref = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll 8
    for (int g = 0; g < kGroups; ++g)
      l += s.part_l[g * kRows + tid] * fast_exp2(s.part_m[g * kRows + tid] - ref);
    s.row_m[tid] = ref;
    s.row_l[tid] = l;
  }
  __syncthreads();
}

// kRows: output rows of a CTA that merges. 512 / D, where a thread has four
// elements and the most parts in flight, for the blocks of few rows, which many
// CTAs share; kMaxRows, for fewer CTAs, for the blocks of up to 128.
template <int D, typename T, int kRows>
__global__ void __launch_bounds__(kThreads)
    tree_finish_kernel(const __grid_constant__ TreeParams p) {
  __shared__ Shared s;
  const int tid = threadIdx.x;
  const int b = blockIdx.z, index = blockIdx.y;
  const int h = index / p.mblocks, mblock = index - h * p.mblocks;
  const int item = (b * p.kv_heads + h) * p.mblocks + mblock;
  // The first CTAs of an item merge its rows; with weights (one block of at most
  // kMaxRows rows) those behind them have each their keys, and all rows.
  const int block = min(p.block_rows, p.rows - mblock * p.block_rows);
  const int mergers = (min(p.block_rows, p.rows) + kRows - 1) / kRows;
  const bool weighs = static_cast<int>(blockIdx.x) >= mergers;
  const int row0 = weighs ? 0 : blockIdx.x * kRows, rows = block - row0;
  const int j = (static_cast<int>(blockIdx.x) - mergers) * kKeysPer + 4 * tid;
  // The lengths and counts are older than the call's first kernel, behind which
  // all of its kernels begin.
  const RowSpan span = row_span(p, b);
  const int n = span.length + span.count, tiles = row_tiles(n);
  const Sharers by = find_place(p, b, index, tiles, s);
  griddep_wait();
  griddep_launch_dependents();
  if (rows <= 0 || (by.count == 1 && !weighs)) return;
  // The scores of the first rows, wherever the row ends: they wait for nothing.
  constexpr int kEarly = 8;
  const float* scores = p.scores + ((int64_t)b * p.kv_heads + h) * p.rows * p.score_stride + j;
  float4 early[kEarly];
  if (weighs && j < p.score_stride) {
#pragma unroll
    for (int r = 0; r < kEarly; ++r)
      if (r < rows) early[r] = *reinterpret_cast<const float4*>(scores + r * p.score_stride);
  }
  const auto* of_rows = reinterpret_cast<const unsigned long long*>(
      p.q_blocks + (int64_t)(item + 1) * p.q_block_bytes - kMaxNodes) - p.block_rows + row0;
  if (tid < min(rows, kMaxRows)) s.masks[tid] = of_rows[tid];
  if (!weighs) {
    // Outputs: a thread has pieces of four elements, neighbours those of the rows.
    constexpr int kMine = kRows * D / 4 / kThreads, kDeep = 8 / kMine;
    float4 o[kMine];
    const int r = tid % kRows, safe_r = min(r, rows - 1);
    int e[kMine];  // first column
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      e[u] = (tid + u * kThreads) / kRows * 4;
    }
    float m[kDeep];
    float4 v[kDeep][kMine];
    auto load = [&](int c0) {
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        const float* x = Parts<D>::of(p, by, min(c0 + i, by.count - 1));
        m[i] = x[row0 + safe_r];
#pragma unroll
        for (int u = 0; u < kMine; ++u)
          v[i][u] =
              *reinterpret_cast<const float4*>(x + Parts<D>::at(p, row0 + safe_r, e[u]));
      }
    };
    load(0);
    join_sums<D, kRows>(p, by, row0, rows, s);
    const float ref = s.row_m[safe_r];
    for (int c0 = 0; c0 < by.count; c0 += kDeep) {
      if (c0 > 0) load(c0);
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        const float f = c0 + i < by.count ? fast_exp2(m[i] - ref) : 0.f;
#pragma unroll
        for (int u = 0; u < kMine; ++u) {
          o[u].x = fmaf(v[i][u].x, f, o[u].x), o[u].y = fmaf(v[i][u].y, f, o[u].y);
          o[u].z = fmaf(v[i][u].z, f, o[u].z), o[u].w = fmaf(v[i][u].w, f, o[u].w);
        }
      }
    }
    if (r < rows) {
      T* out = out_row<T>(p, b, h, mblock * p.block_rows + row0 + r);
#pragma unroll
      for (int u = 0; u < kMine; ++u)
        write_four<T>(out + e[u], s.masks[r] == 0, s.row_l[r], o[u]);
    }
    return;
  }
  join_sums<D, kMaxRows>(p, by, 0, rows, s);
  // A skipped row's nodes have masks of zero: no row of it has weights.
  float* w = p.weights + b * p.w_sb + h * p.w_sh + j;
  float old[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 4; ++u) old[u] = j + u < span.length ? w[u] : 0.f;
  if (tid < rows) {
    const float lse = by.count > 1 ? s.row_m[tid] + log2f(s.row_l[tid])
                                   : p.lse[((int64_t)b * p.kv_heads + h) * p.rows + tid];
    s.row_m[tid] = s.masks[tid] == 0 ? INFINITY : lse;
  }
  bool any = false;
  for (int r = 0; r < rows; ++r) any |= s.masks[r] != 0;
  __syncthreads();
  if (!any || j >= n) return;
  const auto add = [&](const float4& s, float lse) {
    if (lse != INFINITY) {
      sum[0] += fast_exp2(s.x - lse), sum[1] += fast_exp2(s.y - lse);
      sum[2] += fast_exp2(s.z - lse), sum[3] += fast_exp2(s.w - lse);
    }
  };
#pragma unroll
  for (int r = 0; r < kEarly; ++r)
    if (r < rows) add(early[r], s.row_m[r]);
#pragma unroll 8
  for (int r = kEarly; r < rows; ++r)
    add(*reinterpret_cast<const float4*>(scores + r * p.score_stride), s.row_m[r]);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    // A new slot is the node's whose row the first of its query heads is; one
    // without a bit has written none.
    const int node = j + u - span.length;
    if (j + u < n && (node < 0 || s.masks[node * p.group] != 0)) w[u] = old[u] + sum[u];
  }
}

template <int D, typename T, int kRows>
int launch(const TreeParams& p, cudaStream_t stream) {
  unsigned x = (std::min(p.rows, p.block_rows) + kRows - 1) / kRows;
  if (p.weights) x += (p.cache_length + kKeysPer - 1) / kKeysPer;
  return launch_pdl(tree_finish_kernel<D, T, kRows>, dim3(x, p.kv_heads * p.mblocks, p.batch),
                    dim3(kThreads), 0, stream, "tree finish launch", p);
}

template <int D>
int launch(int dtype, const TreeParams& p, cudaStream_t stream) {
  if (dtype == ASRBACK_F32) return launch<D, float, 512 / D>(p, stream);
  return p.block_rows <= kMaxRows ? launch<D, __nv_bfloat16, 512 / D>(p, stream)
                                  : launch<D, __nv_bfloat16, kMaxRows>(p, stream);
}

}  // namespace

namespace tree {

int launch_finish(int dtype, int head_dim, const TreeParams& p, cudaStream_t stream) {
  return head_dim == 64 ? launch<64>(dtype, p, stream) : launch<128>(dtype, p, stream);
}

}  // namespace tree
}  // namespace asrback
