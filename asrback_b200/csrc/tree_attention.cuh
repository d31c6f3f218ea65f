// What the draft-tree attention kernels share: the call's parameters, the
// stretch of the tile list that a CTA works through, and where results go.
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
  int ctas;
  int lead;  // what an item costs a CTA besides its tiles, in tiles
  // The prepared query rows, a block per item: [block rows][D] (bf16: laid out as
  // the products read it, in two parts if rotated), the rows' masks (8 bytes),
  // and kMaxNodes bytes, one per node: its value holds infinities or NaN.
  uint8_t* q_blocks;
  int q_block_bytes;
  float* parts;   // two per CTA: [block rows] m, l, [block rows][D] o
  float* lse;     // with weights: (batch, kv_heads, rows), base 2, of items in one part
  float* scores;  // with weights: (batch, kv_heads, rows, score_stride), base 2
  int64_t score_stride;
  int32_t* status;
};

// A ring's or buffer's place and lap, counted on without divisions.
struct Turn {
  int at = 0, lap = 0;
  __device__ __forceinline__ void next(int size) {
    if (++at == size) at = 0, ++lap;
  }
};

struct RowSpan {
  int length, count;  // cached keys, live nodes; 0, 0 for a row that is skipped
  bool bad;
};

// The row's cached keys and live nodes. A row without nodes reads nothing,
// wherever it stands; a row whose nodes do not fit the cache or the rotary table
// is skipped.
__device__ __forceinline__ RowSpan row_span(const TreeParams& p, int b) {
  const int64_t length = p.lengths[b];
  const int count = p.counts[b];
  const int64_t position = p.q_norm ? p.positions[b] : 0;
  bool bad = count < 0 || count > p.nodes || length < 0 || length > p.cache_length - count;
  if (p.q_norm) bad |= position < 0 || position > p.table_length - count;
  if (bad || count == 0) return {0, 0, bad && count != 0};
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
  int begin;         // unit of the list where the CTA began it
  __device__ __forceinline__ bool whole() const { return tile1 - tile0 == tiles; }
};

// The list of all items' units: `lead` for the item, then one per tile. Every
// CTA takes `per` units.
struct Split {
  int lead, per;
  // With few tiles per CTA their number alone counts.
  __device__ __forceinline__ Split(const TreeParams& p, int tiles) {
    lead = tiles > 4 * p.ctas ? p.lead : 0;
    per = max(1, (tiles + lead * p.batch * p.kv_heads * p.mblocks + p.ctas - 1) / p.ctas);
  }
};

// A CTA's stretch [cur, hi) of the units, from `lo` on: `cur` is unit `unit` of
// item (row, h, mblock). A stretch that ends in an item's lead has none of it.
struct Stretch {
  int lo, hi, cur, lead;
  int row, h, mblock, unit;
  Segment seg;
};

// The CTAs that hold tiles of an item whose units begin at `start` in the list.
struct Sharers {
  int first, count;
  bool begins;  // the item is the first one's first
  __device__ __forceinline__ Sharers(const Split& split, int start, int tiles) {
    const int at = start + split.lead;
    first = at / split.per;
    count = (at + tiles - 1) / split.per - first + 1;
    begins = start <= first * split.per;
  }
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
  const Split split(p, carry);
  const int per_row = p.kv_heads * p.mblocks;
  const int total = carry + split.lead * p.batch * per_row;
  st.lead = split.lead;
  st.lo = static_cast<int>(min(static_cast<int64_t>(blockIdx.x) * split.per, (int64_t)total));
  st.hi = min(st.lo + split.per, total);
  st.cur = st.lo;
  int low = 0, high = p.batch - 1;  // the first row whose units end past lo
  while (low < high) {
    const int mid = (low + high) >> 1;
    if (list.prefix[mid] + split.lead * (mid + 1) * per_row > st.lo) high = mid;
    else low = mid + 1;
  }
  st.row = low;
  const int units =
      row_tiles(static_cast<int>((list.span[low] >> 7) + (list.span[low] & 127u))) + split.lead;
  const int off = st.lo - (low > 0 ? list.prefix[low - 1] + split.lead * low * per_row : 0);
  const int index = off / units;
  st.unit = off - index * units;
  st.h = index / p.mblocks;
  st.mblock = index - st.h * p.mblocks;
  return st;
}

// The next (part of an) item of the stretch; false at its end.
__device__ __forceinline__ bool next_segment(const TreeParams& p, const TileList& list,
                                             Stretch& st) {
  // The end lies `last` tiles into the item.
  const int last = st.unit + st.hi - st.cur - st.lead;
  if (st.cur >= st.hi || last <= 0) return false;
  Segment& s = st.seg;
  s.b = st.row;
  s.h = st.h;
  s.mblock = st.mblock;
  s.item = (s.b * p.kv_heads + s.h) * p.mblocks + s.mblock;
  s.length = static_cast<int>(list.span[s.b] >> 7);
  s.count = static_cast<int>(list.span[s.b] & 127u);
  s.tiles = row_tiles(s.length + s.count);
  s.tile0 = max(st.unit - st.lead, 0);
  s.begin = st.cur;
  s.tile1 = min(s.tiles, last);
  st.cur += s.tile1 + st.lead - st.unit;
  st.unit = 0;
  if (++st.mblock == p.mblocks) {
    st.mblock = 0;
    if (++st.h == p.kv_heads) {
      st.h = 0;
      ++st.row;
    }
  }
  return true;
}

__device__ __forceinline__ float* score_row(const TreeParams& p, const Segment& s, int r) {
  return p.scores + (((int64_t)s.b * p.kv_heads + s.h) * p.rows + r) * p.score_stride;
}

// Where a segment's result goes, if other CTAs hold the rest of its item: m and l
// of the block's rows, then their unnormalised outputs, four columns of all rows
// after the other: the threads of a warp, which have rows, write side by side.
template <int D>
struct Parts {
  __device__ __forceinline__ static int64_t floats(const TreeParams& p) {
    return (int64_t)p.block_rows * (D + 2);
  }
  // Element (row r, column c) of the outputs.
  __device__ __forceinline__ static int at(const TreeParams& p, int r, int c) {
    return 2 * p.block_rows + (c / 4 * p.block_rows + r) * 4 + c % 4;
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
__device__ __forceinline__ T* out_row(const TreeParams& p, int b, int h, int row) {
  return static_cast<T*>(p.out) + b * p.o_sb + (row / p.group) * p.o_sn +
         (h * p.group + row % p.group) * p.o_sh;
}
__device__ __forceinline__ void write_lse(const TreeParams& p, const Segment& s, int row, float m,
                                          float l) {
  p.lse[((int64_t)s.b * p.kv_heads + s.h) * p.rows + row] = m + log2f(l);
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

// Byte offset of 16-byte piece `piece` of row `row` in a tile of `rows` rows of
// D bf16, as a 128-byte-swizzled TMA box lays it out: columns in blocks of 64
// elements, pieces permuted within a row's 128 bytes.
__device__ __forceinline__ int tile_at(int rows, int row, int piece) {
  return (piece >> 3) * rows * 128 + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}

// tree_prepare.cu: the query blocks, and the nodes' keys and values in the
// cache. In bf16 a rotated q is multiplied by the scale and taken in two parts.
int launch_prepare(int dtype, int head_dim, const TreeParams& p, cudaStream_t stream);
// tree_finish.cu: the merge of split items, the accumulated weights.
int launch_finish(int dtype, int head_dim, const TreeParams& p, cudaStream_t stream);
// tree_attention_mma.cu: bf16, one block of 16 query rows, or (head_dim 64) of 32.
int mma_ctas_per_sm(int head_dim, int block_rows);
int launch_mma(int head_dim, const TreeParams& p, cudaStream_t stream);
// tree_attention_tc.cu: bf16, blocks of 32 to 128 query rows.
int launch_tc(int head_dim, const TreeParams& p, cudaStream_t stream);

}  // namespace tree
}  // namespace asrback
