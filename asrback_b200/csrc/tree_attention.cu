// Attention of a tree of drafted tokens over a row's cache, sm_100a: N nodes
// per row (N <= 64; one node is the ordinary decode step, a chain a short
// prompt pass), grouped query heads, lengths read on the device.
//
//   slot(i) = length + i;  keys[slot(i)] = k_i, values[slot(i)] = v_i
//   (with norm weights given, q and k first get their per-head RMSNorm and
//   rotary embedding at position + depth_i)
//   o_i = sum_j p_ij v_j,  p_i = softmax_j(scale q_i . k_j) over the cache's
//   keys j < length and the slots of node i's ancestors (itself among them)
//   weights[j] (optional) += sum_i sum_g p_ij  for j < length, and = for the
//   new slots
//
// Bound. A key and its value are read once and meet N * G query rows (G query
// heads per key/value head): 4 N G D operations per 4 D bytes in bf16, far
// below the tensor cores' 240 operations per byte, so the cache's stream out
// of HBM bounds the call.
//
// Split. The work is the list of 64-key tiles of every (row, key/value head,
// block of query rows); each CTA takes an equal stretch of that list, whatever
// the rows' lengths, so all CTAs stream nearly the same number of bytes. A stretch
// that covers only part of an item leaves its unnormalised result (m, l, o) in
// the workspace. Three launches: tree_prepare.cu writes the nodes' keys and
// values to the cache and the prepared query rows to the workspace (the nodes
// then are an item's last keys, masked by the rows' ancestors), the attention
// (tree_attention_mma.cu or tree_attention_tc.cu in bf16, by the number of query
// rows; below in float32), and tree_finish.cu, which
// merges the parts in list order. Each launch begins while the one before it
// ends; no CTA waits for another, and results do not depend on their order.
#include "../../include/asrback_attn.h"
#include "capi_internal.h"
#include "common.cuh"
#include "tree_attention.cuh"

#include <algorithm>

namespace asrback {
namespace {

using namespace tree;

constexpr int kThreads = 128;

// ------------------------------------------------------------ float32, SIMT
//
// float32 products run on the FMA pipes: a thread takes one key of a tile and
// half the block's rows for the scores, then one column and all rows (head_dim
// 128) or half of them (64) for the output. Few calls have more tiles than the
// GPU takes at once, so a tile's chain of loads and products is what bounds
// them: loads are issued eight at a time, and both products read the operand
// that a warp shares four elements at a time. Measured: 7 rows x 5 nodes of up to
// 448 keys, 6 heads of 64 (one tile per CTA) 13.4 us with what comes before and
// behind, 9.5 of them here.

template <int D>
struct SimtShape {
  static constexpr int kRows = 16;
  static constexpr int kPitch = D + 4;  // floats; spreads a column over the banks
  static constexpr int kOffK = 0;
  static constexpr int kOffV = kTile * kPitch * 4;
  static constexpr int kOffQ = kOffV + kTile * D * 4;
  static constexpr int kOffS = kOffQ + kRows * D * 4;        // scores, then probabilities
  static constexpr int kOffState = kOffS + kRows * kTile * 4;  // m, l, alpha
  static constexpr int kOffO = kOffState + 3 * kRows * 4;
  static constexpr int kOffMasks = kOffO + kRows * D * 4;
  static constexpr int kOffScratch = kOffMasks + kRows * 8;
  static constexpr int kOffList = kOffScratch + 16;
  static constexpr int bytes(int batch) { return kOffList + list_bytes(batch); }
};

template <int D>
__global__ void __launch_bounds__(kThreads)
    tree_simt_kernel(const __grid_constant__ TreeParams p) {
  using Sh = SimtShape<D>;
  constexpr int kRows = Sh::kRows, kPitch = Sh::kPitch;
  constexpr int kHalves = kThreads / D;     // threads per output column
  constexpr int kMine = kRows / kHalves;    // rows per thread in the second product
  extern __shared__ __align__(1024) uint8_t smem[];
  auto* masks = reinterpret_cast<unsigned long long*>(smem + Sh::kOffMasks);
  int* scratch = reinterpret_cast<int*>(smem + Sh::kOffScratch);
  TileList list(smem + Sh::kOffList, p.batch);
  float* ks = reinterpret_cast<float*>(smem + Sh::kOffK);
  float* vs = reinterpret_cast<float*>(smem + Sh::kOffV);
  float* qs = reinterpret_cast<float*>(smem + Sh::kOffQ);
  float* ss = reinterpret_cast<float*>(smem + Sh::kOffS);
  float* state_m = reinterpret_cast<float*>(smem + Sh::kOffState);
  float* state_l = state_m + kRows;
  float* state_a = state_l + kRows;
  float* os = reinterpret_cast<float*>(smem + Sh::kOffO);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  griddep_launch_dependents();
  // The lengths and counts are older than the preparation kernel.
  Stretch st = begin_stretch<kThreads>(p, list, scratch);
  griddep_wait();
  while (next_segment(p, list, st)) {
    const Segment& sg = st.seg;
    const uint8_t* block = p.q_blocks + (int64_t)sg.item * p.q_block_bytes;
    for (int i = tid; i < kRows * D / 4; i += kThreads)
      reinterpret_cast<float4*>(qs)[i] = __ldcg(reinterpret_cast<const float4*>(block) + i);
    if (tid < kRows)
      masks[tid] = __ldcg(reinterpret_cast<const unsigned long long*>(block + kRows * D * 4) + tid);
    if (tid < kRows) state_m[tid] = -INFINITY, state_l[tid] = 0.f;
    // A node whose value holds infinities or NaN: a byte per node, as four words.
    const uint32_t flags =
        __ldcg(reinterpret_cast<const uint32_t*>(block + p.q_block_bytes - kMaxNodes) + lane % 16);
    const bool odd = __any_sync(0xffffffffu, [&] {
      const int live = sg.count - 4 * (lane % 16);  // of the word's nodes
      return live > 0 && (live >= 4 ? flags : flags & ((1u << 8 * live) - 1)) != 0;
    }());
    float o[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) o[i] = 0.f;
    const float* kbase = static_cast<const float*>(p.key_cache) + sg.b * p.c_sb + sg.h * p.c_sh;
    const float* vbase = static_cast<const float*>(p.value_cache) + sg.b * p.c_sb + sg.h * p.c_sh;
    const int total = sg.length + sg.count;
    for (int tile = sg.tile0; tile < sg.tile1 && total > 0; ++tile) {
      const int first_key = tile * kTile, keys = min(kTile, total - first_key);
      const bool edge = first_key + kTile > sg.length;  // nodes in the tile
      __syncthreads();
      constexpr int kBatch = 4, kStep = kThreads / (D / 4);  // rows of a pass
      const int e0 = tid % (D / 4) * 4;
      for (int base = tid / (D / 4); base < kTile; base += kBatch * kStep) {
        float4 k[kBatch], v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int64_t at =
              (int64_t)(first_key + min(base + u * kStep, keys - 1)) * p.c_sp + e0;
          k[u] = *reinterpret_cast<const float4*>(kbase + at);
          v[u] = *reinterpret_cast<const float4*>(vbase + at);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int row = base + u * kStep;
          // Behind the last key: zeros, for the product with zero probabilities.
          if (row >= keys) v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          *reinterpret_cast<float4*>(ks + row * kPitch + e0) = k[u];
          *reinterpret_cast<float4*>(vs + row * D + e0) = v[u];
        }
      }
      __syncthreads();
      {
        const int key = tid % kTile, half = tid / kTile;
        float s[kRows / 2];
#pragma unroll
        for (int i = 0; i < kRows / 2; ++i) s[i] = 0.f;
        for (int e = 0; e < D; e += 4) {
          const float4 k = *reinterpret_cast<const float4*>(ks + key * kPitch + e);
#pragma unroll
          for (int i = 0; i < kRows / 2; ++i) {
            const float4 q =
                *reinterpret_cast<const float4*>(qs + (half * (kRows / 2) + i) * D + e);
            s[i] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[i]))));
          }
        }
#pragma unroll
        for (int i = 0; i < kRows / 2; ++i) {
          const int r = half * (kRows / 2) + i;
          const int age = first_key + key - sg.length;
          const bool seen = key < keys && (age < 0 || (masks[r] >> age & 1) != 0);
          const float x = seen ? s[i] * p.scale_log2 : -INFINITY;
          ss[r * kTile + key] = x;
          if (p.weights && key < keys && r < p.rows) score_row(p, sg, r)[first_key + key] = x;
        }
      }
      __syncthreads();
      for (int r = warp; r < min(kRows, p.rows - sg.mblock * kRows); r += kThreads / 32) {
        const float x0 = ss[r * kTile + lane], x1 = ss[r * kTile + lane + 32];
        float top = fmaxf(x0, x1);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float old = state_m[r], now = fmaxf(old, top), ref = now == -INFINITY ? 0.f : now;
        const float p0 = exp2f(x0 - ref), p1 = exp2f(x1 - ref);
        float sum = p0 + p1;
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        ss[r * kTile + lane] = p0;
        ss[r * kTile + lane + 32] = p1;
        __syncwarp();
        if (lane == 0) {
          const float a = exp2f(old - ref);
          state_m[r] = now;
          state_l[r] = state_l[r] * a + sum;
          state_a[r] = a;
        }
      }
      __syncthreads();
      const int column = tid % D, row0 = tid / D * kMine;
#pragma unroll
      for (int i = 0; i < kMine; ++i) o[i] *= state_a[row0 + i];
      if (!(edge && odd)) {
        for (int key = 0; key < keys; key += 4) {
          float v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = vs[(key + u) * D + column];
#pragma unroll
          for (int i = 0; i < kMine; ++i) {
            const float4 w = *reinterpret_cast<const float4*>(ss + (row0 + i) * kTile + key);
            o[i] = fmaf(w.x, v[0], fmaf(w.y, v[1], fmaf(w.z, v[2], fmaf(w.w, v[3], o[i]))));
          }
        }
      } else {
        // An infinite or NaN value must not reach the nodes that do not see it, as
        // a product with zero would let it.
        for (int key = 0; key < keys; ++key) {
          const float v = vs[key * D + column];
          const int age = first_key + key - sg.length;
#pragma unroll
          for (int i = 0; i < kMine; ++i)
            if (age < 0 || (masks[row0 + i] >> age & 1) != 0)
              o[i] = fmaf(ss[(row0 + i) * kTile + key], v, o[i]);
        }
      }
    }
    __syncthreads();
    const int column = tid % D, row0 = tid / D * kMine;
#pragma unroll
    for (int i = 0; i < kMine; ++i) os[(row0 + i) * D + column] = o[i];
    __syncthreads();
    constexpr int kPieces = D / 4;
    if (sg.whole()) {
      for (int i = tid; i < kRows * kPieces; i += kThreads) {
        const int r = i / kPieces, e = i % kPieces * 4, row = sg.mblock * kRows + r;
        if (row >= p.rows) break;
        write_four<float>(out_row<float>(p, sg.b, sg.h, row) + e, masks[r] == 0, state_l[r],
                          *reinterpret_cast<const float4*>(os + r * D + e));
        if (p.weights && e == 0) write_lse(p, sg, row, state_m[r], state_l[r]);
      }
    } else {
      float* part = Parts<D>::mine(p, st);
      for (int i = tid; i < kRows * kPieces; i += kThreads)
        *reinterpret_cast<float4*>(part + Parts<D>::at(p, i / kPieces, i % kPieces * 4)) =
            reinterpret_cast<const float4*>(os)[i];
      if (tid < kRows) part[tid] = state_m[tid], part[kRows + tid] = state_l[tid];
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ host side

template <int D>
int launch_simt(const TreeParams& p, cudaStream_t stream) {
  // The limit is the largest batch's, set once: one set per call would be another
  // thread's between its set and its launch.
  static thread_local int prepared_device = -1;
  int device = 0;
  if (int rc = check_cuda(cudaGetDevice(&device), "cudaGetDevice")) return rc;
  if (prepared_device != device) {
    if (int rc = check_cuda(cudaFuncSetAttribute(tree_simt_kernel<D>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 SimtShape<D>::bytes(kMaxBatch)),
                            "cudaFuncSetAttribute(tree attention f32)"))
      return rc;
    prepared_device = device;
  }
  return launch_pdl(tree_simt_kernel<D>, dim3(p.ctas), dim3(kThreads),
                    SimtShape<D>::bytes(p.batch), stream, "tree attention (f32) launch", p);
}

// Query rows that one CTA holds against a key tile: blocks of 16 in float32 and for
// the mma.sync kernel, whole warps of TMEM lanes for the tcgen05 kernel.
int rows_per_block(int dtype, int rows) {
  if (dtype == ASRBACK_F32 || rows <= 16) return 16;
  return std::min((rows + 31) / 32 * 32, 128);
}

// In bf16, up to 16 rows per key/value head go to the mma.sync kernel, in head_dim
// 64 up to 32: the tcgen05 kernel's tile has 128 rows whatever it is given, but
// its products cost no registers. Measured, mma.sync and tcgen05: 64 rows of up to
// 1024 keys, 8 heads of 128, 2 query rows 39.6 and 45.3 us, 16 query rows 46.4 and
// 47.5, 32 query rows 60.0 and 51.5 (two parts of 32 queries no longer fit beside
// the outputs); 64 rows of up to 448 keys, 20 heads of 64, 8 query rows 29.3 and
// 53.1 us, 24 query rows 47.3 and 57.2.
bool takes_mma(int dtype, int rows, int head_dim) {
  return dtype == ASRBACK_BF16 && rows <= (head_dim == 64 ? 32 : 16);
}

struct Plan {
  bool mma;
  int block_rows, mblocks, ctas, lead;
  int q_block_bytes;
  size_t q_bytes, part_bytes, lse_bytes, score_bytes;
  int64_t score_stride;
  size_t workspace() const { return q_bytes + part_bytes + lse_bytes + score_bytes; }
};

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

Plan plan_for(int dtype, int batch, int nodes, int heads, int kv_heads, int head_dim,
              int cache_length, bool rotary, bool weights) {
  Plan plan{};
  const int rows = nodes * (heads / kv_heads);
  plan.mma = takes_mma(dtype, rows, head_dim);
  plan.block_rows = rows_per_block(dtype, rows);
  plan.mblocks = (rows + plan.block_rows - 1) / plan.block_rows;
  const int64_t items = (int64_t)batch * kv_heads * plan.mblocks;
  const int64_t tiles = items * ((cache_length + kTile - 1) / kTile);
  // As many CTAs as are resident at once.
  const int per_sm = dtype == ASRBACK_F32 ? (head_dim == 128 ? 2 : 3)
                     : plan.mma ? mma_ctas_per_sm(head_dim, plan.block_rows)
                                : 1;
  plan.ctas = static_cast<int>(std::min<int64_t>(tiles, (int64_t)per_sm * sm_count()));
  // What an item's query block, first scores and end cost a CTA, in tiles, where
  // items are of few tiles. Measured, without and with: 64 rows x 16 nodes of up
  // to 1024 keys (tcgen05) 54.5 and 51.6 us; 64 rows x 8 nodes of up to 448 keys, 20
  // heads of 64 (mma.sync) 32.2 and 30.3 us, but 64 rows x 1 node, 8 heads of
  // 128, whose tiles are twice the bytes, 46.2 and 47.2 us.
  plan.lead = dtype == ASRBACK_F32 ? 0 : !plan.mma ? 2 : head_dim == 64 ? 1 : 0;
  // float32, bf16 as it comes, or (rotary) two bf16 parts; masks and flags.
  const int row_bytes = head_dim * (dtype == ASRBACK_F32 || rotary ? 4 : 2) + 8;
  plan.q_block_bytes = plan.block_rows * row_bytes + kMaxNodes;
  plan.q_bytes = up16((size_t)items * plan.q_block_bytes);
  plan.part_bytes = up16((size_t)2 * plan.ctas * plan.block_rows * (head_dim + 2) * sizeof(float));
  if (weights) {
    plan.score_stride = (cache_length + kTile - 1) / kTile * kTile;
    plan.lse_bytes = up16((size_t)batch * kv_heads * rows * sizeof(float));
    plan.score_bytes = (size_t)batch * kv_heads * rows * plan.score_stride * sizeof(float);
  }
  return plan;
}

}  // namespace
}  // namespace asrback

using namespace asrback;
using namespace asrback::tree;

extern "C" size_t asrback_tree_workspace_bytes(int dtype, int batch, int nodes, int heads,
                                               int kv_heads, int head_dim, int cache_length,
                                               int rotary, int with_weights) {
  if (batch < 1 || nodes < 1 || kv_heads < 1 || heads < kv_heads || head_dim < 1 ||
      cache_length < 1)
    return 0;
  return plan_for(dtype, batch, nodes, heads, kv_heads, head_dim, cache_length, rotary != 0,
                  with_weights != 0)
      .workspace();
}

extern "C" int asrback_tree_attention(
    int dtype, int batch, int nodes, int heads, int kv_heads, int head_dim, int cache_length,
    const void* query, int64_t q_stride_batch, int64_t q_stride_node, int64_t q_stride_head,
    const void* key, int64_t k_stride_batch, int64_t k_stride_node, int64_t k_stride_head,
    const void* value, int64_t v_stride_batch, int64_t v_stride_node, int64_t v_stride_head,
    const void* q_norm_weight, const void* k_norm_weight, float eps, const void* cos,
    const void* sin, int64_t table_stride, int table_length, const int64_t* positions,
    const int64_t* ancestors, const int32_t* depths, const int32_t* counts, const int64_t* lengths,
    void* key_cache, void* value_cache, int64_t c_stride_batch, int64_t c_stride_position,
    int64_t c_stride_head, void* out, int64_t o_stride_batch, int64_t o_stride_node,
    int64_t o_stride_head, float* weights, int64_t w_stride_batch, int64_t w_stride_head,
    float scale, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  if (dtype != ASRBACK_BF16 && dtype != ASRBACK_F32)
    return fail(ASRBACK_ERR_ARGUMENT, "dtype must be ASRBACK_BF16 or ASRBACK_F32, got %d", dtype);
  if (head_dim != 64 && head_dim != 128)
    return fail(ASRBACK_ERR_ARGUMENT, "head_dim must be 64 or 128, got %d", head_dim);
  if (batch < 1 || nodes < 1 || heads < 1 || kv_heads < 1 || cache_length < 1)
    return fail(ASRBACK_ERR_ARGUMENT,
                "batch, nodes, heads, kv_heads and cache length must be positive");
  if (nodes > 64 || batch > kMaxBatch || cache_length > kMaxLength)
    return fail(ASRBACK_ERR_ARGUMENT,
                "at most 64 nodes, %d rows and %d cache positions, got %d, %d and %d", kMaxBatch,
                kMaxLength, nodes, batch, cache_length);
  if (heads % kv_heads != 0)
    return fail(ASRBACK_ERR_ARGUMENT, "heads (%d) must be a multiple of kv_heads (%d)", heads,
                kv_heads);
  if (!query || !key || !value || !key_cache || !value_cache || !out)
    return fail(ASRBACK_ERR_ARGUMENT, "null query, key, value, cache or output pointer");
  if (!ancestors || !depths || !counts || !lengths)
    return fail(ASRBACK_ERR_ARGUMENT, "null ancestors, depths, counts or lengths pointer");
  const bool rotary = q_norm_weight != nullptr;
  if (rotary && (!k_norm_weight || !cos || !sin || !positions || table_length < 1 ||
                 table_stride < head_dim))
    return fail(ASRBACK_ERR_ARGUMENT,
                "q_norm_weight needs k_norm_weight, cos, sin (rows of head_dim) and positions");
  if (!rotary && (k_norm_weight || cos || sin))
    return fail(ASRBACK_ERR_ARGUMENT, "k_norm_weight, cos and sin need q_norm_weight");
  const int64_t esize = dtype == ASRBACK_BF16 ? 2 : 4;
  // Of a dimension of one the stride may be anything: no one reads it.
  const struct { int64_t stride; int size; } strides[] = {
      {q_stride_batch, batch}, {q_stride_node, nodes}, {q_stride_head, heads},
      {k_stride_batch, batch}, {k_stride_node, nodes}, {k_stride_head, kv_heads},
      {v_stride_batch, batch}, {v_stride_node, nodes}, {v_stride_head, kv_heads},
      {c_stride_batch, batch}, {c_stride_position, cache_length}, {c_stride_head, kv_heads},
      {o_stride_batch, batch}, {o_stride_node, nodes}, {o_stride_head, heads}};
  for (const auto& s : strides)
    if (s.size > 1 && (s.stride < 0 || (s.stride * esize) % 16 != 0))
      return fail(ASRBACK_ERR_ARGUMENT,
                  "strides must not be negative and rows must start on 16-byte boundaries");
  if (rotary && (table_stride * esize) % 16 != 0)
    return fail(ASRBACK_ERR_ARGUMENT, "cos and sin rows must start on 16-byte boundaries");
  const void* pointers[] = {query, key, value, key_cache, value_cache, out, q_norm_weight,
                            k_norm_weight, cos, sin};
  for (const void* ptr : pointers)
    if (!aligned16(ptr)) return fail(ASRBACK_ERR_ARGUMENT, "pointers must be 16-byte aligned");
  // The cache and the weights are written: no two of their rows may be one.
  if ((cache_length > 1 && c_stride_position < head_dim) ||
      (kv_heads > 1 && c_stride_head < head_dim) ||
      (batch > 1 && c_stride_batch < head_dim) || (batch > 1 && o_stride_batch < head_dim) ||
      (heads > 1 && o_stride_head < head_dim) || (nodes > 1 && o_stride_node < head_dim))
    return fail(ASRBACK_ERR_ARGUMENT, "cache or output strides do not hold rows of head_dim");
  if (weights && ((batch > 1 && w_stride_batch < cache_length) ||
                  (kv_heads > 1 && w_stride_head < cache_length)))
    return fail(ASRBACK_ERR_ARGUMENT, "weights strides do not hold rows of the cache's length");
  const int rows = nodes * (heads / kv_heads);
  if (weights && rows > kMaxWeightRows)
    return fail(ASRBACK_ERR_ARGUMENT,
                "weights take at most %d query rows per key/value head (nodes x heads / kv_heads), "
                "got %d",
                kMaxWeightRows, rows);
  const Plan plan = plan_for(dtype, batch, nodes, heads, kv_heads, head_dim, cache_length, rotary,
                             weights != nullptr);
  if ((int64_t)batch * kv_heads * plan.mblocks * ((cache_length + kTile - 1) / kTile + plan.lead) >
          (int64_t)1 << 30 ||
      kv_heads * plan.mblocks > 65535)
    return fail(ASRBACK_ERR_ARGUMENT, "too many key tiles or heads for one call");
  const size_t need = plan.workspace();
  if (!workspace || workspace_bytes < need)
    return fail(ASRBACK_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed",
                workspace ? workspace_bytes : (size_t)0, need);
  if (!aligned16(workspace))
    return fail(ASRBACK_ERR_ARGUMENT, "workspace must be 16-byte aligned");

  TreeParams p{};
  p.q = query, p.q_sb = q_stride_batch, p.q_sn = q_stride_node, p.q_sh = q_stride_head;
  p.k = key, p.k_sb = k_stride_batch, p.k_sn = k_stride_node, p.k_sh = k_stride_head;
  p.v = value, p.v_sb = v_stride_batch, p.v_sn = v_stride_node, p.v_sh = v_stride_head;
  p.q_norm = q_norm_weight, p.k_norm = k_norm_weight, p.eps = eps;
  p.cos = cos, p.sin = sin, p.table_stride = table_stride, p.table_length = table_length;
  p.positions = positions, p.ancestors = ancestors, p.depths = depths, p.counts = counts;
  p.lengths = lengths;
  p.key_cache = key_cache, p.value_cache = value_cache;
  p.c_sb = c_stride_batch, p.c_sp = c_stride_position, p.c_sh = c_stride_head;
  p.out = out, p.o_sb = o_stride_batch, p.o_sn = o_stride_node, p.o_sh = o_stride_head;
  p.weights = weights, p.w_sb = w_stride_batch, p.w_sh = w_stride_head;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.batch = batch, p.nodes = nodes, p.kv_heads = kv_heads, p.group = heads / kv_heads;
  p.cache_length = cache_length, p.rows = rows;
  p.block_rows = plan.block_rows, p.mblocks = plan.mblocks;
  p.lead = plan.lead;
  p.ctas = plan.ctas;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  p.q_blocks = at;
  p.q_block_bytes = plan.q_block_bytes;
  at += plan.q_bytes;
  p.parts = reinterpret_cast<float*>(at);
  at += plan.part_bytes;
  p.lse = reinterpret_cast<float*>(at);
  at += plan.lse_bytes;
  p.scores = reinterpret_cast<float*>(at);
  p.score_stride = plan.score_stride;
  p.status = status;

  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc = launch_prepare(dtype, head_dim, p, s);
  if (rc) return rc;
  if (dtype == ASRBACK_BF16)
    rc = plan.mma ? launch_mma(head_dim, p, s) : launch_tc(head_dim, p, s);
  else
    rc = head_dim == 64 ? launch_simt<64>(p, s) : launch_simt<128>(p, s);
  if (!rc) rc = launch_finish(dtype, head_dim, p, s);
  return rc ? rc : ok();
}
