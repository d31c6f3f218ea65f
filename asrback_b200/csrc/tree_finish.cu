// What comes after the draft-tree attention, sm_100a: the items whose tiles lay in
// several CTAs are merged from their parts, and (with weights) the scaled scores
// that the attention left become accumulated weights.
//
// A kernel of its own, so that the attention's CTAs end without waiting for one
// another's parts and the merges run on the whole GPU at once. It moves the parts
// once, 4 bytes per score and 8 per weight, but latency bounds it: a CTA has one
// item, and each of its steps (the item's place in the tile list, the references
// and sums over the parts, the outputs or the scores) loads all it needs at once.
#include "capi_internal.h"
#include "tree_attention.cuh"

#include <algorithm>

namespace asrback {
namespace {

using namespace tree;

constexpr int kThreads = 128;
constexpr int kRowsPer = 16;            // output rows of a CTA
constexpr int kKeysPer = 4 * kThreads;  // keys of a CTA

template <int D, typename T>
__global__ void __launch_bounds__(kThreads)
    tree_finish_kernel(const __grid_constant__ TreeParams p) {
  // [group of parts][row], then the rows' references and sums.
  __shared__ float part_m[kThreads], part_l[kThreads];
  __shared__ float row_m[kRowsPer], row_l[kRowsPer];
  __shared__ unsigned long long masks[kRowsPer];
  const int tid = threadIdx.x;
  const int b = blockIdx.z, index = blockIdx.y;
  const int h = index / p.mblocks, mblock = index - h * p.mblocks;
  const int item = (b * p.kv_heads + h) * p.mblocks + mblock;
  // The CTA's rows. With weights there is one block of at most kRowsPer rows, of
  // which every CTA needs the references, and the first writes the outputs.
  const int row0 = p.weights ? 0 : blockIdx.x * kRowsPer;
  const int rows = min(p.block_rows, p.rows - mblock * p.block_rows) - row0;
  griddep_wait();
  griddep_launch_dependents();
  const int before = b > 0 ? p.place[b - 1] : 0, upto = p.place[b], per = p.place[p.batch];
  const int length = static_cast<int>(p.lengths[b]), count = p.counts[b];
  const auto* of_rows = reinterpret_cast<const unsigned long long*>(
      p.q_blocks + (int64_t)(item + 1) * p.q_block_bytes - kMaxNodes) - p.block_rows + row0;
  if (tid < min(rows, kRowsPer)) masks[tid] = of_rows[tid];
  const int tiles = (upto - before) / (p.kv_heads * p.mblocks);
  const Sharers by(before + index * tiles, tiles, per);
  if (rows <= 0 || (by.count == 1 && !p.weights)) return;
  {
    // References and sums: a thread per row and eighth of the parts.
    constexpr int kGroups = kThreads / kRowsPer, kDeep = 4;
    const int r = tid % kRowsPer, group = tid / kRowsPer;
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
    part_m[tid] = m;
    part_l[tid] = l;
    __syncthreads();
    if (tid < min(rows, kRowsPer)) {
      m = -INFINITY;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) m = fmaxf(m, part_m[g * kRowsPer + tid]);
      const float ref = m == -INFINITY ? 0.f : m;
      l = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        l += part_l[g * kRowsPer + tid] * fast_exp2(part_m[g * kRowsPer + tid] - ref);
      row_m[tid] = ref;
      row_l[tid] = l;
    }
    __syncthreads();
  }
  if (by.count > 1 && (!p.weights || blockIdx.x == 0)) {
    // Outputs: a thread has pieces of four elements.
    constexpr int kPieces = D / 4, kMine = kRowsPer * kPieces / kThreads;
    float4 o[kMine];
    int piece[kMine];  // within the CTA's rows
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      piece[u] = min(tid + u * kThreads, min(rows, kRowsPer) * kPieces - 1);
    }
#pragma unroll 4
    for (int c = 0; c < by.count; ++c) {
      const float* x = Parts<D>::of(p, by, c);
      const float4* y = reinterpret_cast<const float4*>(x + 2 * p.block_rows + row0 * D);
#pragma unroll
      for (int u = 0; u < kMine; ++u) {
        const int r = piece[u] / kPieces;
        const float f = fast_exp2(x[row0 + r] - row_m[r]);
        const float4 v = y[piece[u]];
        o[u].x = fmaf(v.x, f, o[u].x), o[u].y = fmaf(v.y, f, o[u].y);
        o[u].z = fmaf(v.z, f, o[u].z), o[u].w = fmaf(v.w, f, o[u].w);
      }
    }
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      const int r = (tid + u * kThreads) / kPieces, e = piece[u] % kPieces * 4;
      if (r < rows)
        write_four<T>(out_row<T>(p, b, h, mblock * p.block_rows + row0 + r) + e, masks[r] == 0,
                      row_l[r], o[u]);
    }
  }
  if (!p.weights) return;
  // A skipped row's nodes have masks of zero: no row of it has weights.
  __syncthreads();
  if (tid < rows) {
    const float lse = by.count > 1 ? row_m[tid] + log2f(row_l[tid])
                                   : p.lse[((int64_t)b * p.kv_heads + h) * p.rows + tid];
    row_m[tid] = masks[tid] == 0 ? INFINITY : lse;
  }
  bool any = false;
  for (int r = 0; r < rows; ++r) any |= masks[r] != 0;
  __syncthreads();
  const int n = length + count, j = blockIdx.x * kKeysPer + 4 * tid;
  if (!any || j >= n) return;
  const int64_t unit = (int64_t)b * p.kv_heads + h;
  const float* scores = p.scores + unit * p.rows * p.score_stride + j;
  float* w = p.weights + b * p.w_sb + h * p.w_sh + j;
  float old[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 4; ++u) old[u] = j + u < length ? w[u] : 0.f;
#pragma unroll 8
  for (int r = 0; r < rows; ++r) {
    const float4 s = *reinterpret_cast<const float4*>(scores + r * p.score_stride);
    const float lse = row_m[r];
    if (lse != INFINITY) {
      sum[0] += fast_exp2(s.x - lse), sum[1] += fast_exp2(s.y - lse);
      sum[2] += fast_exp2(s.z - lse), sum[3] += fast_exp2(s.w - lse);
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (j + u < n) w[u] = old[u] + sum[u];
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
