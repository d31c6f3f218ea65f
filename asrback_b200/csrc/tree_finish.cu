// What comes after the draft-tree attention, sm_100a: the items whose tiles lay in
// several CTAs are merged from their parts, and (with weights) the scaled scores
// that the attention left become accumulated weights.
//
// A kernel of its own, so that the attention's CTAs end without waiting for one
// another's parts and the merges run on the whole GPU at once. A CTA has one
// item: it first finds the rows' references and sums over the parts (one row per
// thread), then adds up the outputs, or turns its keys' scores into weights and
// adds those up, in row order. It moves the parts once, and 8 bytes per weight
// and 4 per score.
#include "capi_internal.h"
#include "tree_attention.cuh"

#include <algorithm>

namespace asrback {
namespace {

using namespace tree;

constexpr int kThreads = 128;
constexpr int kRowsPer = 16;              // output rows of a CTA
constexpr int kKeysPer = 4 * kThreads;    // keys of a CTA

template <int D, typename T>
__global__ void __launch_bounds__(kThreads)
    tree_finish_kernel(const __grid_constant__ TreeParams p) {
  __shared__ int sums[2][kThreads / 32];
  __shared__ float row_m[128], row_l[128];
  __shared__ unsigned long long masks[128];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.z, index = blockIdx.y;
  const int h = index / p.mblocks, mblock = index - h * p.mblocks;
  const int item = (b * p.kv_heads + h) * p.mblocks + mblock;
  const int rows = min(p.block_rows, p.rows - mblock * p.block_rows);
  griddep_wait();
  griddep_launch_dependents();
  // The item's place in the tile list.
  int before = 0, total = 0;
  for (int i = tid; i < p.batch; i += kThreads) {
    const RowSpan s = row_span(p, i);
    const int tiles = row_tiles(s.length + s.count) * p.kv_heads * p.mblocks;
    total += tiles;
    before += i < b ? tiles : 0;
  }
  const RowSpan span = row_span(p, b);
  const auto* of_rows = reinterpret_cast<const unsigned long long*>(
      p.q_blocks + (int64_t)(item + 1) * p.q_block_bytes - kMaxNodes) - p.block_rows;
  if (tid < rows) masks[tid] = of_rows[tid];
  before = __reduce_add_sync(0xffffffffu, before);
  total = __reduce_add_sync(0xffffffffu, total);
  if (lane == 0) sums[0][warp] = before, sums[1][warp] = total;
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) before += sums[0][w], total += sums[1][w];
  const int tiles = row_tiles(span.length + span.count);
  const Sharers by(before + index * tiles, tiles, stretch_tiles(p, total));
  if (by.count > 1) {
    // References and sums: kDeep parts' loads in flight.
    constexpr int kDeep = 8;
    if (tid < rows) {
      float m = -INFINITY, l = 0.f;
      for (int c0 = 0; c0 < by.count; c0 += kDeep) {
        float m2[kDeep], l2[kDeep];
#pragma unroll
        for (int c = 0; c < kDeep; ++c) {
          const bool in = c0 + c < by.count;
          const float* x = Parts<D>::of(p, by, in ? c0 + c : 0);
          m2[c] = in ? x[tid] : -INFINITY;
          l2[c] = in ? x[p.block_rows + tid] : 0.f;
        }
#pragma unroll
        for (int c = 0; c < kDeep; ++c) {
          const float now = fmaxf(m, m2[c]), ref = now == -INFINITY ? 0.f : now;
          l = l * fast_exp2(m - ref) + l2[c] * fast_exp2(m2[c] - ref);
          m = now;
        }
      }
      row_m[tid] = m == -INFINITY ? 0.f : m;
      row_l[tid] = l;
    }
    __syncthreads();
    // Outputs of kRowsPer rows: a thread has pieces of four elements.
    constexpr int kPieces = D / 4, kMine = kRowsPer * kPieces / kThreads;
    const int row0 = blockIdx.x * kRowsPer;
    if (row0 < rows) {
      float4 o[kMine];
      int piece[kMine];
#pragma unroll
      for (int u = 0; u < kMine; ++u) {
        o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        piece[u] = min(row0 * kPieces + tid + u * kThreads, rows * kPieces - 1);
      }
#pragma unroll 4
      for (int c = 0; c < by.count; ++c) {
        const float* x = Parts<D>::of(p, by, c);
#pragma unroll
        for (int u = 0; u < kMine; ++u) {
          const int r = piece[u] / kPieces;
          const float f = fast_exp2(x[r] - row_m[r]);
          const float4 y = reinterpret_cast<const float4*>(x + 2 * p.block_rows)[piece[u]];
          o[u].x = fmaf(y.x, f, o[u].x), o[u].y = fmaf(y.y, f, o[u].y);
          o[u].z = fmaf(y.z, f, o[u].z), o[u].w = fmaf(y.w, f, o[u].w);
        }
      }
#pragma unroll
      for (int u = 0; u < kMine; ++u) {
        const int r = row0 + (tid + u * kThreads) / kPieces, e = piece[u] % kPieces * 4;
        if (r < rows)
          write_four<T>(out_row<T>(p, b, h, mblock * p.block_rows + r) + e, masks[r] == 0,
                        row_l[r], o[u]);
      }
    }
  }
  if (!p.weights || span.count == 0) return;
  // Weights: one block of at most kMaxWeightRows rows per head here.
  __syncthreads();
  if (tid < rows) {
    const float lse = by.count > 1 ? row_m[tid] + log2f(row_l[tid])
                                   : p.lse[((int64_t)b * p.kv_heads + h) * p.rows + tid];
    row_m[tid] = masks[tid] == 0 ? INFINITY : lse;  // an empty row has no weights
  }
  __syncthreads();
  const int n = span.length + span.count;
  const int64_t unit = (int64_t)b * p.kv_heads + h;
#pragma unroll
  for (int u = 0; u < kKeysPer / kThreads; ++u) {
    const int j = blockIdx.x * kKeysPer + u * kThreads + tid;
    if (j >= n) break;
    float sum = 0.f;
#pragma unroll 4
    for (int r = 0; r < rows; ++r)
      if (row_m[r] != INFINITY)
        sum += fast_exp2(p.scores[(unit * p.rows + r) * p.score_stride + j] - row_m[r]);
    float* w = p.weights + b * p.w_sb + h * p.w_sh + j;
    *w = j < span.length ? *w + sum : sum;
  }
}

template <int D, typename T>
int launch(const TreeParams& p, cudaStream_t stream) {
  unsigned x = (std::min(p.rows, p.block_rows) + kRowsPer - 1) / kRowsPer;
  if (p.weights) x = std::max<unsigned>(x, (p.cache_length + kKeysPer - 1) / kKeysPer);
  return launch_pdl(tree_finish_kernel<D, T>, dim3(x, p.kv_heads * p.mblocks, p.batch),
                    dim3(kThreads), 0, stream, "tree finish launch", p);
}

}  // namespace

namespace tree {

int launch_finish(int dtype, int head_dim, const TreeParams& p, cudaStream_t stream) {
  if (dtype == ASRBACK_F32)
    return head_dim == 64 ? launch<64, float>(p, stream) : launch<128, float>(p, stream);
  return head_dim == 64 ? launch<64, __nv_bfloat16>(p, stream)
                        : launch<128, __nv_bfloat16>(p, stream);
}

}  // namespace tree
}  // namespace asrback
