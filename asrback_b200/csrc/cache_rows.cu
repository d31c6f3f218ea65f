// Rows of a key/value cache moved to the front of their batch row: the commit
// of a draft tree's accepted nodes and the eviction of keys by accumulated
// attention weight, sm_100a.
//
// Both move cache row source[k] to row target + k with source ascending and
// source[k] >= k, in place. A move then never overwrites a row that a later
// move reads, so rows are moved in ascending order, a batch of loads before
// its stores, with no copy of the cache. A moved row is read once and written
// once. Measured: the commit of 64 rows x 16 nodes over 28 layers of 8 heads of 128
// 6 us, which launch and load latency bound (its 14 MB keep DRAM 9 % busy); an
// eviction of 64 rows from 1024 slots to 512, 8 heads of 128, 52 us, near HBM's
// stream: 273 MB to read and write at 5.2 TB/s, of which part stays in L2 (cold and
// profiled 216 MB in 49 us, DRAM 54 % busy); of 2 rows from 16384 slots to 4096 29
// us, 12 for the selection and 16 for the moves, bound by their barriers and
// latencies (DRAM 1 and 24 % busy).
#include "../../include/asrback_attn.h"
#include "capi_internal.h"
#include "common.cuh"

#include <algorithm>

namespace asrback {
namespace {

struct CacheView {
  uint8_t* base;  // strides in bytes
  int64_t layer, batch, position, head;
};

// -------------------------------------------------------------------- commit

struct CommitParams {
  CacheView cache[2];  // keys, values
  int layers, batch, heads, length, vectors;  // vectors: 16-byte pieces of a head's row
  const int32_t* path;
  const int32_t* counts;
  const int64_t* start;
  int nodes;
  float* weights;  // or null
  int64_t w_layer, w_batch, w_head;
  int32_t* status;
};

constexpr int kMaxNodes = 64;
constexpr int kCommitThreads = 128;

// A thread owns one 16-byte column of the moved rows and moves it node by
// node, eight loads in flight. A row of the batch accepts a few nodes of some
// kilobytes over every layer, so the columns are what there is to spread out.
__global__ void __launch_bounds__(kCommitThreads)
    commit_kernel(const __grid_constant__ CommitParams p) {
  __shared__ int path[kMaxNodes];
  __shared__ int moved[2];  // first node that moves, one past the last
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.y, layer = blockIdx.z >> 1, which = blockIdx.z & 1;
  const int column = blockIdx.x * kCommitThreads + threadIdx.x;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const int count = p.counts[b];
    const int64_t start = p.start[b];
    int node[2];
    bool bad = count < 0 || count > p.nodes;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = lane + 32 * u;
      node[u] = k < p.nodes ? p.path[(int64_t)b * p.nodes + k] : -1;
      path[k] = node[u];
    }
    __syncwarp();
    uint64_t moves = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = lane + 32 * u;
      if (k < count && k < p.nodes) {
        const int before = k > 0 ? path[k - 1] : -1;
        bad |= node[u] <= before || node[u] >= p.nodes || start < 0 ||
               start >= p.length - node[u];  // no sum that could pass 63 bits
      }
      moves |= static_cast<uint64_t>(__ballot_sync(0xffffffffu, k < count && node[u] != k))
               << (32 * u);
    }
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
      if (bad && p.status) atomicOr(p.status, ASRBACK_STATUS_POSITION);
      moved[0] = bad || moves == 0 ? 0 : __ffsll(static_cast<long long>(moves)) - 1;
      moved[1] = bad || moves == 0 ? 0 : count;
    }
  }
  __syncthreads();
  const int first = moved[0], last = moved[1];
  if (first >= last) return;
  const int64_t start = p.start[b];
  if (which == 0 && p.weights) {
    for (int h = column; h < p.heads; h += gridDim.x * kCommitThreads) {
      float* row = p.weights + layer * p.w_layer + b * p.w_batch + h * p.w_head + start;
      for (int k = first; k < last; ++k) row[k] = row[path[k]];
    }
  }
  if (column >= p.heads * p.vectors) return;
  const CacheView& c = p.cache[which];
  uint8_t* rows = c.base + layer * c.layer + b * c.batch + (column / p.vectors) * c.head +
                  start * c.position + (column % p.vectors) * 16;
  for (int k = first; k < last; k += 8) {
    uint4 piece[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (k + u < last) piece[u] = *reinterpret_cast<const uint4*>(rows + path[k + u] * c.position);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (k + u < last) *reinterpret_cast<uint4*>(rows + (k + u) * c.position) = piece[u];
  }
}

// --------------------------------------------------------- eviction: selection

struct SelectParams {
  float* weights;
  int64_t w_layer, w_batch, w_head;
  const int64_t* lengths;
  int64_t* new_lengths;
  int32_t* kept;  // (layers, batch, heads, budget)
  int batch, heads, length, budget, sink, recent;
  int cluster;  // CTAs that share a row
  int32_t* status;
};

constexpr int kSelectThreads = 256;
constexpr int kShortRow = 4 * kSelectThreads;  // slots that one CTA holds in registers

// What lies at `at` in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ int load_remote(const int* at, int rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];"
               : "=r"(v)
               : "r"(cluster_map(smem_addr(at), rank))
               : "memory");
  return v;
}

// Order-preserving key of a weight: larger weight, larger key. Zeros of both
// signs are equal, NaN counts as -inf. The protected slots' key is above every
// weight's.
constexpr uint32_t kProtected = 0xffffffffu;
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  if (w == 0.f) w = 0.f;
  const uint32_t u = __float_as_uint(w);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// A cluster of CTAs per (layer, row, head) finds the `budget` largest keys, each
// CTA in a contiguous share of the slots. The threshold (the budget-th largest
// key) is built digit by digit from the top: the keys that share the digits so
// far are counted by their next one, every CTA adds up the cluster's counts, and
// the digit in which the budget-th lies is the threshold's. It ends early once
// the keys down to that digit are exactly the budget. Keys equal to the threshold
// are taken from the lowest slot up. A thread holds V slots of a chunk in
// registers, kSelectThreads apart; a share of one chunk is read once. The kept
// weights are compacted here, their slots go to `kept`.
//
// The counting's instructions bound it, not the bytes (one SM took 18 us for a
// row of 16384 keys), hence the clusters.
//
// kMoves: two CTAs (a cluster) select for a row of one chunk, each for itself; the
// slots also go to `own_kept`, in shared memory, and only the first one writes.
// Returns whether the row is cut.
template <int V, bool kCluster, bool kMoves>
__device__ __forceinline__ bool select_row(const SelectParams& p, int* own_kept) {
  constexpr int kChunk = kSelectThreads * V, kWarps = kSelectThreads / 32;
  constexpr int kBits = 8, kDigits = 32 / kBits, kBins = 1 << kBits;
  static_assert(kBins == kSelectThreads, "a thread per bin");
  __shared__ int bins[kDigits][kBins];
  __shared__ int found[3];          // the digit, the keys above it, its own
  __shared__ int scan[V * kWarps];  // keys above | equal << 16 of each 32 slots, in slot order
  __shared__ int sums[kWarps];
  __shared__ int share[2];  // of this CTA: keys above, equal
  const int cluster = kCluster ? p.cluster : 1, ctas = kMoves ? 2 : cluster;
  const int h = blockIdx.x / ctas, rank = kMoves ? 0 : blockIdx.x - h * ctas;
  const bool writes = !kMoves || blockIdx.x % 2 == 0;
  const int b = blockIdx.y, layer = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t given = p.lengths[b];
  const bool first = h == 0 && layer == 0 && rank == 0 && tid == 0 && writes;
  int32_t* kept = p.kept + (((int64_t)layer * p.batch + b) * p.heads + h) * p.budget;
  const int every = cluster * kSelectThreads, mine = rank * kSelectThreads + tid;
  if (given < 0 || given > p.length) {
    if (first) {
      p.new_lengths[b] = given;
      if (p.status) atomicOr(p.status, ASRBACK_STATUS_POSITION);
    }
    for (int k = mine; k < p.budget && writes; k += every) kept[k] = -1;
    return false;
  }
  const int n = static_cast<int>(given);
  if (first) p.new_lengths[b] = min(n, p.budget);
  if (n <= p.budget) {
    for (int k = mine; k < p.budget && writes; k += every) kept[k] = k < n ? k : -1;
    return false;
  }
  float* row = p.weights + layer * p.w_layer + b * p.w_batch + h * p.w_head;
  // Rows of more than one chunk per CTA come to clusters only.
  const int chunks = kCluster ? (n + cluster * kChunk - 1) / (cluster * kChunk) : 1;
  const int start = rank * chunks * kChunk, tail = n - p.recent;
  float raw[V];
  uint32_t key[V];
  // Slots past the row's end hold key 0, below every weight's.
  auto load = [&](int chunk) {
    const int base = start + chunk * kChunk + tid;
#pragma unroll
    for (int u = 0; u < V; ++u) raw[u] = row[min(base + u * kSelectThreads, n - 1)];
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int j = base + u * kSelectThreads;
      key[u] = j >= n ? 0u : j < p.sink || j >= tail ? kProtected : weight_key(raw[u]);
    }
  };
  auto barrier = [&] {
    if constexpr (kCluster) cluster_sync();
    else __syncthreads();
  };
#pragma unroll
  for (int d = 0; d < kDigits; ++d) bins[d][tid] = 0;
  load(0);
  __syncthreads();
  uint32_t threshold = 0;
  int ties = p.budget;  // kept keys that share the threshold's digits so far
  bool exact = false;
  for (int d = 0; d < kDigits && !exact; ++d) {
    // Bits [low, low + kBits) of the keys that share the threshold's above them.
    const int low = 32 - (d + 1) * kBits;
    for (int chunk = 0; chunk < chunks; ++chunk) {
      if (chunks > 1) load(chunk);
#pragma unroll
      for (int u = 0; u < V; ++u) {
        const bool in =
            key[u] != 0u && static_cast<uint64_t>(key[u] ^ threshold) >> (low + kBits) == 0;
        const int bin = key[u] >> low & (kBins - 1);
        // Many equal keys, as zeros are, count at once.
        const uint32_t ins = __ballot_sync(0xffffffffu, in);
        if (ins == 0) continue;
        const int leader = __ffs(ins) - 1;
        const int leaders = __shfl_sync(0xffffffffu, bin, leader);  // every lane takes part
        const bool same = in && bin == leaders;
        const uint32_t sames = __ballot_sync(0xffffffffu, same);
        if (lane == leader) atomicAdd(&bins[d][bin], __popc(sames));
        else if (in && !same) atomicAdd(&bins[d][bin], 1);
      }
    }
    barrier();
    const int mine_bin = kBins - 1 - tid;
    int own = 0;
    if constexpr (kCluster) {
      for (int r = 0; r < cluster; ++r) own += load_remote(&bins[d][mine_bin], r);
    } else {
      own = bins[d][mine_bin];
    }
    int through = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, through, o);
      if (lane >= o) through += x;
    }
    if (lane == 31) sums[warp] = through;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (w < warp) through += sums[w];
    if (through - own < ties && ties <= through)
      found[0] = mine_bin, found[1] = through - own, found[2] = own;
    __syncthreads();
    threshold |= static_cast<uint32_t>(found[0]) << low;
    ties -= found[1];
    exact = ties == found[2];
  }
  if (exact) ties = n;  // whatever shares the digits found is kept
  // Each 32 slots' keys above and equal, and what lies before them in the chunk;
  // returns the chunk's.
  auto count = [&] {
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const uint32_t above = __ballot_sync(0xffffffffu, key[u] > threshold);
      const uint32_t equal = __ballot_sync(0xffffffffu, key[u] == threshold);
      if (lane == 0) scan[u * kWarps + warp] = __popc(above) | __popc(equal) << 16;
    }
    __syncthreads();  // all counts are there; the chunk's raw weights have been read
    int own = 0, through = 0;
    if (tid < V * kWarps) {
      own = through = scan[tid];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, through, o);
        if (lane >= o) through += x;
      }
      if (lane == 31) sums[warp] = through;
    }
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < V * kWarps / 32; ++w) {
      if (w < warp) through += sums[w];
      all += sums[w];
    }
    if (tid < V * kWarps) scan[tid] = through - own;
    __syncthreads();
    return all;
  };
  int above_before = 0, equal_before = 0;  // of the slots before the chunk
  if constexpr (kCluster) {
    int above = 0, equal = 0;
    for (int chunk = 0; chunk < chunks; ++chunk) {
      if (chunks > 1) load(chunk);
      const int all = count();
      above += all & 0xffff, equal += all >> 16;
    }
    if (tid == 0) share[0] = above, share[1] = equal;
    barrier();
    for (int r = 0; r < rank; ++r)
      above_before += load_remote(&share[0], r), equal_before += load_remote(&share[1], r);
  }
  const uint32_t lower = (1u << lane) - 1;
  for (int chunk = 0; chunk < chunks; ++chunk) {
    if (chunks > 1) load(chunk);
    const int all = kCluster && chunks == 1 ? 0 : count();
    if constexpr (kMoves) cluster_sync();  // both CTAs have read the weights
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const bool over = key[u] > threshold, same = key[u] == threshold;
      const uint32_t above = __ballot_sync(0xffffffffu, over);
      const uint32_t equal = __ballot_sync(0xffffffffu, same);
      const int at = scan[u * kWarps + warp];
      const int above_at = above_before + (at & 0xffff) + __popc(above & lower);
      const int equal_at = equal_before + (at >> 16) + __popc(equal & lower);
      if (over || (same && equal_at < ties)) {
        const int k = above_at + min(equal_at, ties);
        const int slot = start + chunk * kChunk + u * kSelectThreads + tid;
        if constexpr (kMoves) own_kept[k] = slot;
        if (writes) kept[k] = slot;
        // All CTAs have read the row, if it is of one chunk each.
        if (writes && chunks == 1) row[k] = raw[u];
      }
    }
    above_before += all & 0xffff;
    equal_before += all >> 16;
    __syncthreads();  // `scan` and `sums` have been read
  }
  if (chunks > 1) {
    // In turns from the front, whose loads come before their stores: what a turn
    // writes lies before all that later turns read.
    barrier();
    for (int k0 = 0; k0 < p.budget; k0 += every) {
      const int k = k0 + mine;
      const float w = k < p.budget ? row[kept[k]] : 0.f;
      barrier();
      if (k < p.budget) row[k] = w;
    }
  }
  if constexpr (kCluster) cluster_sync();  // the others have read this CTA's counts
  return true;
}

template <int V, bool kCluster>
__global__ void __launch_bounds__(kSelectThreads)
    select_kernel(const __grid_constant__ SelectParams p) {
  griddep_wait();
  griddep_launch_dependents();
  select_row<V, kCluster, false>(p, nullptr);
}

// -------------------------------------------------------- eviction: the moves

struct MoveParams {
  CacheView cache[2];
  const int64_t* lengths;
  const int32_t* kept;
  int batch, heads, length, budget;
  int vectors;  // 16-byte pieces of the part of a row that one CTA moves
  int cluster;  // CTAs that move one head's rows
};

constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 4;

// Moves the part of one head's kept rows that lies at `rows`, kMoveUnroll rows per
// thread and turn of `cluster` CTAs. A turn's loads come before its barrier and
// its stores after it; the next turn's loads are issued in between, since its
// rows lie behind all that this turn writes.
template <typename Barrier>
__device__ __forceinline__ void move_rows(uint8_t* rows, int64_t position, const int32_t* kept,
                                          int budget, int vectors, int rank, int cluster,
                                          Barrier barrier) {
  const int lanes = kMoveThreads / vectors;  // rows per pass of the CTA
  const int turn = lanes * kMoveUnroll * cluster;
  const int mine = rank * lanes * kMoveUnroll + threadIdx.x / vectors;
  uint4 piece[2][kMoveUnroll];
  int from[2][kMoveUnroll];
  auto load = [&](int set, int k0) {
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int k = k0 + u * lanes + mine;
      from[set][u] = k < budget ? kept[k] : k;
    }
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int k = k0 + u * lanes + mine;
      if (from[set][u] != k)
        piece[set][u] = *reinterpret_cast<const uint4*>(rows + from[set][u] * position);
    }
  };
  auto store = [&](int set, int k0) {
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int k = k0 + u * lanes + mine;
      if (from[set][u] != k) *reinterpret_cast<uint4*>(rows + k * position) = piece[set][u];
    }
  };
  load(0, 0);
  for (int k0 = 0; k0 < budget; k0 += 2 * turn) {
    load(1, k0 + turn);
    barrier();
    store(0, k0);
    load(0, k0 + 2 * turn);
    barrier();
    store(1, k0 + turn);
  }
}

// A cluster of CTAs moves one head's kept rows of the keys or of the values (or a
// part of their columns).
template <bool kCluster>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ MoveParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int cluster = kCluster ? p.cluster : 1;
  const int h = blockIdx.x / cluster, rank = blockIdx.x - h * cluster;
  const int b = blockIdx.y % p.batch, layer = blockIdx.y / p.batch;
  const int which = blockIdx.z & 1, part = blockIdx.z >> 1;
  const int64_t given = p.lengths[b];
  if (given <= p.budget || given > p.length) return;
  const CacheView& c = p.cache[which];
  uint8_t* rows = c.base + layer * c.layer + b * c.batch + h * c.head +
                  (part * p.vectors + threadIdx.x % p.vectors) * 16;
  const int32_t* kept = p.kept + ((int64_t)blockIdx.y * p.heads + h) * p.budget;
  move_rows(rows, c.position, kept, p.budget, p.vectors, rank, cluster, [] {
    if constexpr (kCluster) cluster_sync();
    else __syncthreads();
  });
}

// Selection and moves in one, for many short rows: a cluster of two CTAs per
// (layer, row, head), one for the keys and one for the values, so that some rows'
// counting runs beside others' moves.
__global__ void __launch_bounds__(kMoveThreads)
    evict_kernel(const __grid_constant__ SelectParams p, const __grid_constant__ MoveParams m) {
  static_assert(kMoveThreads == kSelectThreads);
  __shared__ int kept[kShortRow];
  griddep_wait();
  griddep_launch_dependents();
  if (!select_row<kShortRow / kSelectThreads, false, true>(p, kept)) return;
  __syncthreads();
  const CacheView& c = m.cache[blockIdx.x % 2];
  uint8_t* rows = c.base + blockIdx.z * c.layer + blockIdx.y * c.batch +
                  (blockIdx.x / 2) * c.head + threadIdx.x % m.vectors * 16;
  move_rows(rows, c.position, kept, m.budget, m.vectors, 0, 1, [] { __syncthreads(); });
}

// Rows of weights that are written: no two of them may be one.
int check_weights(int layers, int batch, int heads, int length, int64_t layer, int64_t row,
                  int64_t head) {
  if ((layers > 1 && layer < length) || (batch > 1 && row < length) || (heads > 1 && head < length))
    return fail(ASRBACK_ERR_ARGUMENT, "weights strides do not hold rows of the cache's length");
  return ASRBACK_OK;
}

// Checks a cache's shape and fills `view` (strides in bytes); an ABI code.
int cache_view(CacheView* view, const char* name, void* base, int64_t esize, int layers, int rows,
               int head_dim, int64_t layer, int64_t batch, int64_t position, int64_t head) {
  if (!base) return fail(ASRBACK_ERR_ARGUMENT, "null %s pointer", name);
  if (!aligned16(base) || (layer * esize) % 16 || (batch * esize) % 16 ||
      (position * esize) % 16 || (head * esize) % 16)
    return fail(ASRBACK_ERR_ARGUMENT,
                "%s rows must start on 16-byte boundaries (pointer and strides)", name);
  if (position < head_dim || head < head_dim || (layers > 1 && layer < head_dim) ||
      (rows > 1 && batch < head_dim))
    return fail(ASRBACK_ERR_ARGUMENT, "%s strides do not hold rows of head_dim elements", name);
  *view = {static_cast<uint8_t*>(base), layer * esize, batch * esize, position * esize,
           head * esize};
  return ASRBACK_OK;
}

int check_cache_sizes(int dtype, int layers, int batch, int heads, int head_dim, int length) {
  if (dtype != ASRBACK_BF16 && dtype != ASRBACK_F32)
    return fail(ASRBACK_ERR_ARGUMENT, "dtype must be ASRBACK_BF16 or ASRBACK_F32, got %d", dtype);
  if (layers < 1 || batch < 1 || heads < 1 || length < 1)
    return fail(ASRBACK_ERR_ARGUMENT, "layers, batch, heads and cache length must be positive");
  if (head_dim != 64 && head_dim != 128)
    return fail(ASRBACK_ERR_ARGUMENT, "head_dim must be 64 or 128, got %d", head_dim);
  return ASRBACK_OK;
}

}  // namespace
}  // namespace asrback

using namespace asrback;

extern "C" int asrback_commit_tree(int dtype, int layers, int batch, int nodes, int heads,
                                   int head_dim, int length, void* key_cache, void* value_cache,
                                   int64_t c_stride_layer, int64_t c_stride_batch,
                                   int64_t c_stride_position, int64_t c_stride_head, float* weights,
                                   int64_t w_stride_layer, int64_t w_stride_batch,
                                   int64_t w_stride_head, const int32_t* path,
                                   const int32_t* counts, const int64_t* start, int32_t* status,
                                   void* stream) {
  if (int rc = check_cache_sizes(dtype, layers, batch, heads, head_dim, length)) return rc;
  if (nodes < 1 || nodes > kMaxNodes)
    return fail(ASRBACK_ERR_ARGUMENT, "nodes must be in [1, %d], got %d", kMaxNodes, nodes);
  if (batch > 65535 || layers > 32767)
    return fail(ASRBACK_ERR_ARGUMENT, "at most 65535 rows and 32767 layers, got %d and %d", batch,
                layers);
  if (!path || !counts || !start)
    return fail(ASRBACK_ERR_ARGUMENT, "null path, counts or start pointer");
  if (weights)
    if (int rc = check_weights(layers, batch, heads, length, w_stride_layer, w_stride_batch,
                               w_stride_head))
      return rc;
  const int64_t esize = dtype == ASRBACK_BF16 ? 2 : 4;
  CommitParams p{};
  if (int rc = cache_view(&p.cache[0], "key_cache", key_cache, esize, layers, batch, head_dim,
                          c_stride_layer, c_stride_batch, c_stride_position, c_stride_head))
    return rc;
  if (int rc = cache_view(&p.cache[1], "value_cache", value_cache, esize, layers, batch, head_dim,
                          c_stride_layer, c_stride_batch, c_stride_position, c_stride_head))
    return rc;
  p.layers = layers;
  p.batch = batch;
  p.heads = heads;
  p.length = length;
  p.vectors = static_cast<int>(head_dim * esize / 16);
  p.path = path;
  p.counts = counts;
  p.start = start;
  p.nodes = nodes;
  p.weights = weights;
  p.w_layer = w_stride_layer;
  p.w_batch = w_stride_batch;
  p.w_head = w_stride_head;
  p.status = status;
  const unsigned columns = (heads * p.vectors + kCommitThreads - 1) / kCommitThreads;
  if (int rc = launch_pdl(commit_kernel, dim3(columns, batch, 2 * layers), dim3(kCommitThreads), 0,
                          static_cast<cudaStream_t>(stream), "commit launch", p))
    return rc;
  return ok();
}

extern "C" int asrback_evict(int dtype, int layers, int batch, int heads, int head_dim, int length,
                             void* key_cache, void* value_cache, int64_t c_stride_layer,
                             int64_t c_stride_batch, int64_t c_stride_position,
                             int64_t c_stride_head, float* weights, int64_t w_stride_layer,
                             int64_t w_stride_batch, int64_t w_stride_head, const int64_t* lengths,
                             int budget, int sink, int recent, int64_t* new_lengths, int32_t* kept,
                             int32_t* status, void* stream) {
  if (int rc = check_cache_sizes(dtype, layers, batch, heads, head_dim, length)) return rc;
  if (budget < 1 || budget > length)
    return fail(ASRBACK_ERR_ARGUMENT, "budget must be in [1, cache length %d], got %d", length,
                budget);
  if (sink < 0 || recent < 0 || sink > budget - recent)
    return fail(ASRBACK_ERR_ARGUMENT,
                "sink and recent must not be negative and at most budget together");
  if (static_cast<int64_t>(layers) * batch > 65535 || layers > 65535 || batch > 65535)
    return fail(ASRBACK_ERR_ARGUMENT, "at most 65535 rows over all layers, got %d x %d", layers,
                batch);
  if (!weights || !lengths || !new_lengths || !kept)
    return fail(ASRBACK_ERR_ARGUMENT, "null weights, lengths, new_lengths or kept pointer");
  if (new_lengths == lengths)
    return fail(ASRBACK_ERR_ARGUMENT, "new_lengths must not be lengths, which is read meanwhile");
  if (int rc = check_weights(layers, batch, heads, length, w_stride_layer, w_stride_batch,
                             w_stride_head))
    return rc;
  const int64_t esize = dtype == ASRBACK_BF16 ? 2 : 4;
  MoveParams m{};
  if (int rc = cache_view(&m.cache[0], "key_cache", key_cache, esize, layers, batch, head_dim,
                          c_stride_layer, c_stride_batch, c_stride_position, c_stride_head))
    return rc;
  if (int rc = cache_view(&m.cache[1], "value_cache", value_cache, esize, layers, batch, head_dim,
                          c_stride_layer, c_stride_batch, c_stride_position, c_stride_head))
    return rc;
  SelectParams s{};
  s.weights = weights;
  s.w_layer = w_stride_layer;
  s.w_batch = w_stride_batch;
  s.w_head = w_stride_head;
  s.lengths = lengths;
  s.new_lengths = new_lengths;
  s.kept = kept;
  s.batch = batch;
  s.heads = heads;
  s.length = length;
  s.budget = budget;
  s.sink = sink;
  s.recent = recent;
  s.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  m.lengths = lengths;
  m.kept = kept;
  m.batch = batch;
  m.heads = heads;
  m.length = length;
  m.budget = budget;
  m.vectors = static_cast<int>(head_dim * esize / 16);
  const int64_t moves = static_cast<int64_t>(layers) * batch * heads * 2;
  int rc;
  // One launch where two CTAs per row fill the GPU: 64 rows of 8 heads from 1024
  // slots to 512 54 us, 59 in two launches. Fewer rows want more CTAs each.
  if (length <= kShortRow && moves >= 2 * sm_count()) {
    rc = launch_pdl_cluster(evict_kernel, dim3(heads * 2, batch, layers), dim3(kMoveThreads), 0, 2,
                            st, "evict launch", s, m);
    return rc ? rc : ok();
  }
  if (length <= kShortRow) {
    rc = launch_pdl(select_kernel<4, false>, dim3(heads, batch, layers), dim3(kSelectThreads), 0, st,
                    "evict selection launch", s);
  } else {
    // As many CTAs as hold a row's slots in registers, up to 8.
    s.cluster = 2;
    while (s.cluster < 8 && s.cluster * 8 * kSelectThreads < length) s.cluster *= 2;
    rc = launch_pdl_cluster(select_kernel<8, true>, dim3(heads * s.cluster, batch, layers),
                            dim3(kSelectThreads), 0, s.cluster, st, "evict selection launch", s);
  }
  if (rc) return rc;
  // A head's rows are split over a cluster until the launch has four CTAs per SM
  // or a turn of the cluster holds all rows; then their columns, in parts of at
  // least 64 bytes, until it has two. (2 rows from 16384 slots to 4096: 43 us
  // with neither, 36 with clusters, 31.5 with both.)
  int rows_per_turn = kMoveThreads / m.vectors * kMoveUnroll;
  m.cluster = 1;
  while (m.cluster < 8 && moves * m.cluster < 4 * sm_count() && rows_per_turn * m.cluster < budget)
    m.cluster *= 2;
  int parts = 1;
  while (m.vectors > 4 && moves * m.cluster * parts < 2 * sm_count() &&
         rows_per_turn * m.cluster < budget)
    m.vectors /= 2, parts *= 2, rows_per_turn *= 2;
  const dim3 move_grid(heads * m.cluster, layers * batch, 2 * parts);
  if (m.cluster == 1)
    rc = launch_pdl(move_kernel<false>, move_grid, dim3(kMoveThreads), 0, st, "evict move launch",
                    m);
  else
    rc = launch_pdl_cluster(move_kernel<true>, move_grid, dim3(kMoveThreads), 0, m.cluster, st,
                            "evict move launch", m);
  return rc ? rc : ok();
}
