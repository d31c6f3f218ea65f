// Trees of drafted tokens: the plan that every layer's attention shares, and
// the greedy acceptance walk with the decode-state update, sm_100a.
//
// Both kernels give a row of the batch to one warp. A row has at most 64
// nodes, so a lane holds two, a node's ancestors are the bits of one 64-bit
// word, and nothing crosses a warp. The kernels move a few hundred bytes per
// row: they are bound by launch and load latency, so each input is loaded
// once, all loads in flight together, before the first is used. Measured, 64 rows
// x 16 nodes: 1.7 and 2.9 us.
#include "../../include/asrback_attn.h"
#include "capi_internal.h"
#include "common.cuh"

namespace asrback {
namespace {

constexpr int kMaxNodes = 64;
constexpr int kMaxEos = 8;
constexpr int kWarps = 4;  // rows per CTA: 1 to 64 rows spread over the SMs

// ------------------------------------------------------------------- the plan

// ancestors[i] = {i} + ancestors[parent i], depths[i] = depths[parent i] + 1.
// Pointer jumping: after round r a node has joined its 2^r nearest ancestors,
// so six rounds reach all 64 whatever the tree's shape.
__global__ void __launch_bounds__(kWarps * 32)
    draft_tree_kernel(int batch, int nodes, const int32_t* __restrict__ parents,
                      int64_t parents_stride, const int32_t* __restrict__ counts,
                      const int64_t* __restrict__ lengths, int64_t capacity,
                      int64_t* __restrict__ ancestors, int32_t* __restrict__ depths,
                      int32_t* __restrict__ live_counts, int32_t* status) {
  __shared__ unsigned long long mask[kWarps][kMaxNodes];
  __shared__ int jump[kWarps][kMaxNodes], depth[kWarps][kMaxNodes];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x * kWarps + warp;
  griddep_wait();
  griddep_launch_dependents();
  if (b >= batch) return;
  int count = counts ? counts[b] : nodes;
  const int64_t length = lengths ? lengths[b] : 0;
  int parent[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    parent[u] = i < nodes ? parents[b * parents_stride + i] : -1;
  }
  bool bad = count < 0 || count > nodes;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    bad |= i < count && (parent[u] < -1 || parent[u] >= i);
  }
  if (__any_sync(0xffffffffu, bad)) {
    count = 0;
    if (lane == 0 && status) atomicOr(status, ASRBACK_STATUS_TREE);
  }
  // The first nodes are a tree by themselves, since parents come before children.
  if (lengths && count > 0) {
    const int64_t room = length < 0 || length >= capacity ? 0 : capacity - length;
    if (room == 0 && lane == 0 && status) atomicOr(status, ASRBACK_STATUS_POSITION);
    count = room < count ? static_cast<int>(room) : count;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    const bool live = i < count;
    mask[warp][i] = live ? 1ull << i : 0ull;
    jump[warp][i] = live ? parent[u] : -1;
    depth[warp][i] = live && parent[u] >= 0 ? 1 : 0;
  }
  __syncwarp();
  for (int round = 0; round < 6; ++round) {
    unsigned long long m[2];
    int to[2], d[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = lane + 32 * u, at = jump[warp][i];
      m[u] = mask[warp][i] | (at >= 0 ? mask[warp][at] : 0ull);
      d[u] = depth[warp][i] + (at >= 0 ? depth[warp][at] : 0);
      to[u] = at >= 0 ? jump[warp][at] : -1;
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = lane + 32 * u;
      mask[warp][i] = m[u];
      depth[warp][i] = d[u];
      jump[warp][i] = to[u];
    }
    __syncwarp();
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    if (i < nodes) {
      ancestors[(int64_t)b * nodes + i] = static_cast<int64_t>(mask[warp][i]);
      depths[(int64_t)b * nodes + i] = depth[warp][i];
    }
  }
  if (lane == 0) live_counts[b] = count;
}

// ------------------------------------------------------------- the acceptance

struct AcceptParams {
  int batch, nodes, n_eos;
  const int32_t* parents;
  int64_t parents_stride;
  const int32_t* counts;
  const int64_t* drafts;
  const int64_t* chosen;
  const float* logprob;
  int64_t drafts_stride, chosen_stride, logprob_stride;
  int64_t* tokens;
  int64_t tokens_stride;
  int64_t* position;
  const int64_t* end;
  uint8_t* finished;
  float* sum_logprobs;
  int64_t* generated;
  int64_t generated_stride, generated_cols;
  int64_t* lengths;
  int32_t* path;
  int32_t* accepted;
  int64_t* start;
  int32_t* status;
  int64_t eos[kMaxEos];
};

// The walk of a row: from node 0, emit the token chosen there, then step to
// the lowest child that holds that token, until there is none or the row ends
// (EOS, or its position reaches `end`). Every node finds whether it matches
// its parent's token at once, so that the walk itself is one shared-memory
// read per step. The log-probabilities are added in the walk's order, which
// makes the sum the one that as many single steps give.
__global__ void __launch_bounds__(kWarps * 32)
    accept_tree_kernel(const __grid_constant__ AcceptParams p) {
  __shared__ int next[kWarps][kMaxNodes], taken[kWarps][kMaxNodes];
  __shared__ int64_t chosen[kWarps][kMaxNodes];
  __shared__ float logprob[kWarps][kMaxNodes];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x * kWarps + warp;
  griddep_wait();
  griddep_launch_dependents();
  if (b >= p.batch) return;
  int count = p.counts[b];
  const int64_t position = p.position[b], end = p.end[b];
  const bool done = p.finished[b] != 0;
  const int64_t start = p.lengths ? p.lengths[b] : position;
  float sum = p.sum_logprobs[b];
  int parent[2];
  int64_t draft[2], token[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    const bool in = i < p.nodes;
    parent[u] = in ? p.parents[b * p.parents_stride + i] : -1;
    draft[u] = in ? p.drafts[b * p.drafts_stride + i] : 0;
    token[u] = in ? p.chosen[b * p.chosen_stride + i] : 0;
    chosen[warp][i] = token[u];
    logprob[warp][i] = in ? p.logprob[b * p.logprob_stride + i] : 0.f;
    next[warp][i] = kMaxNodes;
    taken[warp][i] = -1;
  }
  bool bad = count < 0 || count > p.nodes;
  uint64_t stops = 0;  // nodes whose chosen token is an end of sequence
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    bad |= i < count && (parent[u] < -1 || parent[u] >= i);
    bool eos = false;
    for (int e = 0; e < p.n_eos; ++e) eos |= token[u] == p.eos[e];
    stops |= static_cast<uint64_t>(__ballot_sync(0xffffffffu, eos)) << (32 * u);
  }
  if (__any_sync(0xffffffffu, bad)) {
    count = 0;
    if (lane == 0 && p.status) atomicOr(p.status, ASRBACK_STATUS_TREE);
  }
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    if (i < count && parent[u] >= 0 && draft[u] == chosen[warp][parent[u]])
      atomicMin(&next[warp][parent[u]], i);
  }
  __syncwarp();
  // Every lane walks the same nodes; lane 0 notes them.
  int steps = 0, last = 0;
  bool over = done;
  if (!done && count > 0) {
    const int64_t room = end - position;  // the row ends behind its room-th token
    int at = 0;
    while (true) {
      last = at;
      if (lane == 0) taken[warp][steps] = at;
      sum += logprob[warp][at];
      ++steps;
      over = (stops >> at & 1) != 0 || steps >= room;
      at = next[warp][at];
      if (over || at >= kMaxNodes) break;
    }
  }
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int k = lane + 32 * u;
    if (k >= p.nodes) break;
    const int node = taken[warp][k];
    p.path[(int64_t)b * p.nodes + k] = node;
    if (k < steps) {
      const int64_t at = position + 1 + k;
      if (at >= 0 && at < p.generated_cols) {
        p.generated[b * p.generated_stride + at] = chosen[warp][node];
      } else if (p.status) {
        atomicOr(p.status, ASRBACK_STATUS_POSITION);
      }
    }
  }
  if (lane == 0) {
    p.accepted[b] = steps;
    p.start[b] = start;
    if (steps > 0) {
      p.tokens[b * p.tokens_stride] = chosen[warp][last];
      p.position[b] = position + steps;
      p.sum_logprobs[b] = sum;
      p.finished[b] = over;
      if (p.lengths) p.lengths[b] = start + steps;
    }
  }
}

}  // namespace
}  // namespace asrback

using namespace asrback;

extern "C" int asrback_draft_tree_in_cache(int batch, int nodes, const int32_t* parents,
                                           int64_t parents_stride, const int32_t* counts,
                                           const int64_t* lengths, int64_t capacity,
                                           int64_t* ancestors, int32_t* depths,
                                           int32_t* live_counts, int32_t* status, void* stream) {
  if (batch < 1 || nodes < 1 || nodes > kMaxNodes)
    return fail(ASRBACK_ERR_ARGUMENT, "batch must be positive and nodes in [1, %d], got %d and %d",
                kMaxNodes, batch, nodes);
  if (!parents || !ancestors || !depths || !live_counts)
    return fail(ASRBACK_ERR_ARGUMENT, "null parents, ancestors, depths or live_counts pointer");
  if (parents_stride < 0 || (parents_stride > 0 && parents_stride < nodes))
    return fail(ASRBACK_ERR_ARGUMENT,
                "parents_stride must be 0 (one tree for every row) or at least nodes");
  if (lengths && capacity < 1)
    return fail(ASRBACK_ERR_ARGUMENT, "capacity must be positive where lengths are given");
  if (int rc = launch_pdl(draft_tree_kernel, dim3((batch + kWarps - 1) / kWarps), dim3(kWarps * 32),
                          0, static_cast<cudaStream_t>(stream), "draft tree launch", batch, nodes,
                          parents, parents_stride, counts, lengths, capacity, ancestors, depths,
                          live_counts, status))
    return rc;
  return ok();
}

extern "C" int asrback_draft_tree(int batch, int nodes, const int32_t* parents,
                                  int64_t parents_stride, const int32_t* counts,
                                  int64_t* ancestors, int32_t* depths, int32_t* live_counts,
                                  int32_t* status, void* stream) {
  return asrback_draft_tree_in_cache(batch, nodes, parents, parents_stride, counts, nullptr, 0,
                                     ancestors, depths, live_counts, status, stream);
}

extern "C" int asrback_accept_tree(
    int batch, int nodes, const int32_t* parents, int64_t parents_stride, const int32_t* counts,
    const int64_t* drafts, int64_t drafts_stride, const int64_t* chosen, int64_t chosen_stride,
    const float* logprob, int64_t logprob_stride, int64_t* tokens, int64_t tokens_stride,
    int64_t* position, const int64_t* end, uint8_t* finished, float* sum_logprobs,
    int64_t* generated, int64_t generated_stride, int64_t generated_cols, int64_t* lengths,
    const int64_t* eos_ids, int n_eos, int32_t* path, int32_t* accepted, int64_t* start,
    int32_t* status, void* stream) {
  if (batch < 1 || nodes < 1 || nodes > kMaxNodes)
    return fail(ASRBACK_ERR_ARGUMENT, "batch must be positive and nodes in [1, %d], got %d and %d",
                kMaxNodes, batch, nodes);
  if (!parents || !counts || !drafts || !chosen || !logprob)
    return fail(ASRBACK_ERR_ARGUMENT, "null parents, counts, drafts, chosen or logprob pointer");
  if (!tokens || !position || !end || !finished || !sum_logprobs || !generated)
    return fail(ASRBACK_ERR_ARGUMENT, "null decode state pointer");
  if (!path || !accepted || !start)
    return fail(ASRBACK_ERR_ARGUMENT, "null path, accepted or start pointer");
  if (parents_stride < 0 || (parents_stride > 0 && parents_stride < nodes))
    return fail(ASRBACK_ERR_ARGUMENT,
                "parents_stride must be 0 (one tree for every row) or at least nodes");
  if (drafts_stride < nodes || chosen_stride < nodes || logprob_stride < nodes)
    return fail(ASRBACK_ERR_ARGUMENT, "row strides must be at least nodes");
  if (tokens_stride < 1 || generated_cols < 1 || generated_stride < generated_cols)
    return fail(ASRBACK_ERR_ARGUMENT,
                "tokens_stride and generated_cols must be positive, generated_stride at least "
                "generated_cols");
  if (n_eos < 0 || n_eos > kMaxEos || (n_eos > 0 && !eos_ids))
    return fail(ASRBACK_ERR_ARGUMENT, "n_eos must be in [0, %d] with eos_ids given", kMaxEos);
  AcceptParams p{};
  p.batch = batch;
  p.nodes = nodes;
  p.parents = parents;
  p.parents_stride = parents_stride;
  p.counts = counts;
  p.drafts = drafts;
  p.drafts_stride = drafts_stride;
  p.chosen = chosen;
  p.chosen_stride = chosen_stride;
  p.logprob = logprob;
  p.logprob_stride = logprob_stride;
  p.tokens = tokens;
  p.tokens_stride = tokens_stride;
  p.position = position;
  p.end = end;
  p.finished = finished;
  p.sum_logprobs = sum_logprobs;
  p.generated = generated;
  p.generated_stride = generated_stride;
  p.generated_cols = generated_cols;
  p.lengths = lengths;
  p.path = path;
  p.accepted = accepted;
  p.start = start;
  p.status = status;
  p.n_eos = n_eos;
  for (int e = 0; e < n_eos; ++e) p.eos[e] = eos_ids[e];
  if (int rc = launch_pdl(accept_tree_kernel, dim3((batch + kWarps - 1) / kWarps),
                          dim3(kWarps * 32), 0, static_cast<cudaStream_t>(stream),
                          "accept tree launch", p))
    return rc;
  return ok();
}
