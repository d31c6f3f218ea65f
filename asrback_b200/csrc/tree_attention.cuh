// What the draft-tree attention kernels share: the call's parameters, the
// stretch of the tile list that a CTA works through, and the end of a segment
// (output, or part and merge).
#pragma once

#include "common.cuh"

namespace asrback {
namespace tree {

constexpr int kTile = 64;            // keys per tile
constexpr int kMaxNodes = 64;
constexpr int kMaxBatch = 1024;      // rows whose tile counts fit the CTA's shared memory
constexpr int kMaxWeightRows = 16;   // query rows per key/value head of a call with weights
constexpr int kMaxLength = 1 << 24;  // cache positions (packed with the node count)

struct TreeParams {
  const void *q, *k, *v;  // element strides: row of the batch, node, head
  int64_t q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh;
  const void *q_norm, *k_norm, *cos, *sin;  // all null: no norm, no rotary embedding
  float eps;
  int64_t table_stride;
  int table_length;
  const int64_t *positions, *ancestors, *lengths;
  const int32_t *depths, *counts;
  void *key_cache, *value_cache;
  int64_t c_sb, c_sp, c_sh;
  void* out;
  int64_t o_sb, o_sn, o_sh;
  float* weights;
  int64_t w_sb, w_sh;
  float scale_log2;  // softmax scale times log2(e)
  int batch, nodes, kv_heads, group, cache_length;
  int rows, block_rows, mblocks;  // query rows per key/value head, in blocks
  int ctas, min_tiles;            // fewest tiles of a CTA's stretch
  // The prepared query rows, a block per item: [block rows][D] (bf16: laid out as
  // the products read it, in two parts if rotated), then the rows' masks.
  uint8_t* q_blocks;
  int q_block_bytes;
  int* counters;  // one per item, zero between calls
  float* parts;   // two per CTA: [block rows] m, l, [block rows][D] o
  float* lse;     // with weights: (batch, kv_heads, rows), base 2, +inf for an empty row
  float* scores;  // with weights: (batch, kv_heads, rows, score_stride), base 2
  int64_t score_stride;
  int32_t* status;
};

struct RowSpan {
  int length, count;  // cached keys, live nodes; 0, 0 for a row that is skipped
  bool bad;
};

// The row's cached keys and live nodes. A row without nodes reads nothing; a
// row whose nodes do not fit the cache or the rotary table is skipped.
__device__ __forceinline__ RowSpan row_span(const TreeParams& p, int b) {
  const int64_t length = p.lengths[b];
  const int count = p.counts[b];
  const int64_t position = p.q_norm ? p.positions[b] : 0;
  bool bad = count < 0 || count > p.nodes || length < 0 || length > p.cache_length - count;
  if (p.q_norm) bad |= position < 0 || position > p.table_length - count;
  if (bad || count == 0) return {0, 0, bad};
  return {static_cast<int>(length), count, false};
}

// Tiles over the row's keys, the tree's behind the cached ones; a row that is
// skipped has one, for its zeros.
__device__ __forceinline__ int row_tiles(int keys) { return max(1, (keys + kTile - 1) / kTile); }

// The tile list of the call, in the CTA's shared memory: list_bytes(batch) at
// `prefix`, the spans behind the prefix.
struct TileList {
  int* prefix;     // tiles of rows 0..b
  uint32_t* span;  // length << 7 | count
  __device__ __forceinline__ TileList(uint8_t* at, int batch)
      : prefix(reinterpret_cast<int*>(at)), span(reinterpret_cast<uint32_t*>(at) + batch) {}
};
__host__ __device__ constexpr int list_bytes(int batch) { return (8 * batch + 15) / 16 * 16; }

struct Segment {
  int b, h, mblock, item;
  int length, count;
  int tiles;         // of the item
  int tile0, tile1;  // this segment's
  int begin;         // tile0 in the list of all tiles
  __device__ __forceinline__ bool whole() const { return tile1 - tile0 == tiles; }
};

// A CTA's stretch [cur, hi) of the list of all items' tiles, `per` tiles each
// from `lo` on: `cur` is tile `tile` of item (row, h, mblock).
struct Stretch {
  int lo, hi, cur, per;
  int row, h, mblock, tile;
  Segment seg;
};

// Fills the tile list and finds the CTA's stretch. All kThreads threads of the
// CTA call it; `scratch` holds kThreads / 32 ints.
template <int kThreads>
__device__ __forceinline__ Stretch begin_stretch(const TreeParams& p, const TileList& list,
                                                 int* scratch) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int carry = 0;
  for (int base = 0; base < p.batch; base += kThreads) {
    const int b = base + tid;
    int tiles = 0;
    if (b < p.batch) {
      const RowSpan s = row_span(p, b);
      list.span[b] = static_cast<uint32_t>(s.length) << 7 | s.count;
      tiles = row_tiles(s.length + s.count) * p.kv_heads * p.mblocks;
    }
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    sum += carry;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      const int s = scratch[w];
      if (w < warp) sum += s;
      carry += s;
    }
    if (b < p.batch) list.prefix[b] = sum;
    __syncthreads();
  }
  Stretch st;
  const int total = carry;
  st.per = max((total + p.ctas - 1) / p.ctas, p.min_tiles);
  st.lo = static_cast<int>(min(static_cast<int64_t>(blockIdx.x) * st.per, (int64_t)total));
  st.hi = min(st.lo + st.per, total);
  st.cur = st.lo;
  int low = 0, high = p.batch - 1;  // the first row whose prefix lies past lo
  while (low < high) {
    const int mid = (low + high) >> 1;
    if (list.prefix[mid] > st.lo) high = mid;
    else low = mid + 1;
  }
  st.row = low;
  const int tiles = row_tiles(static_cast<int>((list.span[low] >> 7) + (list.span[low] & 127u)));
  const int off = st.lo - (low > 0 ? list.prefix[low - 1] : 0), index = off / tiles;
  st.tile = off - index * tiles;
  st.h = index / p.mblocks;
  st.mblock = index - st.h * p.mblocks;
  return st;
}

// The next (part of an) item of the stretch; false at its end.
__device__ __forceinline__ bool next_segment(const TreeParams& p, const TileList& list,
                                             Stretch& st) {
  if (st.cur >= st.hi) return false;
  Segment& s = st.seg;
  s.b = st.row;
  s.h = st.h;
  s.mblock = st.mblock;
  s.item = (s.b * p.kv_heads + s.h) * p.mblocks + s.mblock;
  s.length = static_cast<int>(list.span[s.b] >> 7);
  s.count = static_cast<int>(list.span[s.b] & 127u);
  s.tiles = row_tiles(s.length + s.count);
  s.tile0 = st.tile;
  s.begin = st.cur;
  s.tile1 = min(s.tiles, s.tile0 + st.hi - st.cur);
  st.cur += s.tile1 - s.tile0;
  st.tile = 0;
  if (++st.mblock == p.mblocks) {
    st.mblock = 0;
    if (++st.h == p.kv_heads) {
      st.h = 0;
      ++st.row;
    }
  }
  return true;
}

// The CTAs that hold parts of the segment's item.
struct Sharers {
  int first, count;
  bool begins;  // the item begins the first one's stretch
  __device__ __forceinline__ Sharers(const Stretch& st) {
    const int start = st.seg.begin - st.seg.tile0;
    first = start / st.per;
    count = (start + st.seg.tiles - 1) / st.per - first + 1;
    begins = start == first * st.per;
  }
};

__device__ __forceinline__ float* score_row(const TreeParams& p, const Segment& s, int r) {
  return p.scores + (((int64_t)s.b * p.kv_heads + s.h) * p.rows + r) * p.score_stride;
}

// Where a segment's result goes, if other CTAs hold the rest of its item: m and l
// of the block's rows, then their unnormalised outputs.
template <int D>
struct Parts {
  __device__ __forceinline__ static int64_t floats(const TreeParams& p) {
    return (int64_t)p.block_rows * (D + 2);
  }
  // A CTA's first segment leaves part 0, a later one (its last) part 1.
  __device__ __forceinline__ static float* mine(const TreeParams& p, const Stretch& st) {
    return p.parts + (2 * blockIdx.x + (st.seg.begin == st.lo ? 0 : 1)) * floats(p);
  }
  // Part c of the item; its first CTA may have begun it behind another item.
  __device__ __forceinline__ static const float* of(const TreeParams& p, const Sharers& by, int c) {
    return p.parts + (2 * (by.first + c) + (c == 0 && !by.begins ? 1 : 0)) * floats(p);
  }
};

// An output row's elements from `e` on, and its log-sum-exp (with weights).
template <typename T>
__device__ __forceinline__ T* out_row(const TreeParams& p, const Segment& s, int row) {
  return static_cast<T*>(p.out) + s.b * p.o_sb + (row / p.group) * p.o_sn +
         (s.h * p.group + row % p.group) * p.o_sh;
}
__device__ __forceinline__ void write_lse(const TreeParams& p, const Segment& s, int row,
                                          bool empty, float m, float l) {
  p.lse[((int64_t)s.b * p.kv_heads + s.h) * p.rows + row] = empty ? INFINITY : m + log2f(l);
}

// Four elements of a row from its unnormalised sum; zeros for an empty row.
template <typename T>
__device__ __forceinline__ void write_four(T* out, bool empty, float l, float4 o) {
  const float f = 1.f / l;
  o = empty ? make_float4(0.f, 0.f, 0.f, 0.f)
            : make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(out) = o;
  } else {
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(o.x, o.y), __floats2bfloat162_rn(o.z, o.w)};
    *reinterpret_cast<uint2*>(out) = *reinterpret_cast<uint2*>(h);
  }
}

// Merges the item's parts, in the order of the tile list, and writes its rows
// out; kThreads threads (all of a group that `sync` joins) call it, after the
// item's last ticket. First a thread per row finds the row's reference and sum,
// then the outputs are added up, kDeep loads in flight per thread. `rows_m` and
// `rows_l` hold a float per row of the block.
template <int D, int kThreads, typename T, typename Sync>
__device__ __forceinline__ void merge_parts(const TreeParams& p, const Segment& s,
                                            const Sharers& by, const unsigned long long* masks,
                                            float* rows_m, float* rows_l, int tid, Sync sync) {
  constexpr int kPieces = D / 4, kDeep = 4;
  const int ctas = by.count;
  const int rows = min(p.block_rows, p.rows - s.mblock * p.block_rows);
  for (int r = tid; r < rows; r += kThreads) {
    float m = -INFINITY, l = 0.f;
    for (int c0 = 0; c0 < ctas; c0 += kDeep) {
      float m2[kDeep], l2[kDeep];
#pragma unroll
      for (int c = 0; c < kDeep; ++c) {
        const bool in = c0 + c < ctas;
        const float* x = Parts<D>::of(p, by, in ? c0 + c : 0);
        m2[c] = in ? __ldcg(x + r) : -INFINITY;
        l2[c] = in ? __ldcg(x + p.block_rows + r) : 0.f;
      }
#pragma unroll
      for (int c = 0; c < kDeep; ++c) {
        const float now = fmaxf(m, m2[c]), ref = now == -INFINITY ? 0.f : now;
        l = l * fast_exp2(m - ref) + l2[c] * fast_exp2(m2[c] - ref);
        m = now;
      }
    }
    rows_m[r] = m == -INFINITY ? 0.f : m;
    rows_l[r] = l;
    if (p.weights) write_lse(p, s, s.mblock * p.block_rows + r, masks[r] == 0, m, l);
  }
  sync();
  // Parts lie a fixed distance apart but for the first.
  const float* first = Parts<D>::of(p, by, 0);
  const float* second = Parts<D>::of(p, by, 1);
  const int64_t step = 2 * Parts<D>::floats(p);
  const int body = 2 * p.block_rows;
  for (int at0 = tid; at0 < rows * kPieces; at0 += kDeep * kThreads) {
    float4 o[kDeep];
    float m[kDeep];
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      m[u] = rows_m[min(at0 + u * kThreads, rows * kPieces - 1) / kPieces];
    }
    const float* x = first;
#pragma unroll 2
    for (int c = 0; c < ctas; ++c) {
      float4 y[kDeep];
      float a[kDeep];
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const int at = min(at0 + u * kThreads, rows * kPieces - 1);
        a[u] = __ldcg(x + at / kPieces);
        y[u] = __ldcg(reinterpret_cast<const float4*>(x + body + 4 * at));
      }
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const float f = fast_exp2(a[u] - m[u]);
        o[u].x = fmaf(y[u].x, f, o[u].x), o[u].y = fmaf(y[u].y, f, o[u].y);
        o[u].z = fmaf(y[u].z, f, o[u].z), o[u].w = fmaf(y[u].w, f, o[u].w);
      }
      x = c == 0 ? second : x + step;
    }
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int at = at0 + u * kThreads, r = at / kPieces, e = at % kPieces * 4;
      if (at >= rows * kPieces) break;
      write_four<T>(out_row<T>(p, s, s.mblock * p.block_rows + r) + e, masks[r] == 0, rows_l[r],
                    o[u]);
    }
  }
}

// Takes a ticket of the item (one thread, once its CTA's part is in memory):
// true for the last of the item's CTAs, which also re-arms the counter.
__device__ __forceinline__ bool take_ticket(const Sharers& by, int* counter) {
  const bool last = atomicAdd(counter, 1) == by.count - 1;
  if (last) *counter = 0;
  return last;
}

// Byte offset of 16-byte piece `piece` of row `row` in a tile of `rows` rows of
// D bf16, as a 128-byte-swizzled TMA box lays it out: columns in blocks of 64
// elements, pieces permuted within a row's 128 bytes.
__device__ __forceinline__ int tile_at(int rows, int row, int piece) {
  return (piece >> 3) * rows * 128 + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}

// tree_prepare.cu: the query blocks, and the nodes' keys and values in the
// cache. In bf16 a rotated q is multiplied by the scale and taken in two parts.
int launch_prepare(int dtype, int head_dim, const TreeParams& p, cudaStream_t stream);
// tree_attention_tc.cu: bf16.
int launch_tc(int head_dim, const TreeParams& p, cudaStream_t stream);

}  // namespace tree
}  // namespace asrback
