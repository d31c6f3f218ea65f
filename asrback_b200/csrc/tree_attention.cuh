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
  int batch, nodes, kv_heads, group, rows, mblocks, cache_length, ctas;
  // The prepared query rows, a block per item: kQParts x [block rows][D]
  // (bf16: laid out as the products read it), then the rows' masks.
  uint8_t* q_blocks;
  int q_block_bytes;
  int* counters;  // per item and group of 16 rows, zero between calls
  float* parts;   // two per CTA: [rows] m, [rows] l, [rows][D] o
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
  int first_cta, last_cta;
};

// A CTA's stretch [lo, hi) of the list of all items' tiles, `per` tiles each.
struct Stretch {
  int lo, hi, cur, per, row;
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
  st.per = (total + p.ctas - 1) / p.ctas;
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
  return st;
}

// The next (part of an) item of the stretch; false at its end.
__device__ __forceinline__ bool next_segment(const TreeParams& p, const TileList& list,
                                             Stretch& st) {
  if (st.cur >= st.hi) return false;
  while (list.prefix[st.row] <= st.cur) ++st.row;
  Segment& s = st.seg;
  const int base = st.row > 0 ? list.prefix[st.row - 1] : 0;
  s.b = st.row;
  s.length = static_cast<int>(list.span[s.b] >> 7);
  s.count = static_cast<int>(list.span[s.b] & 127u);
  s.tiles = row_tiles(s.length + s.count);
  const int index = (st.cur - base) / s.tiles;
  s.h = index / p.mblocks;
  s.mblock = index % p.mblocks;
  s.item = s.b * p.kv_heads * p.mblocks + index;
  const int start = base + index * s.tiles;
  s.tile0 = st.cur - start;
  s.tile1 = min(s.tiles, st.hi - start);
  s.first_cta = start / st.per;
  s.last_cta = (start + s.tiles - 1) / st.per;
  s.begin = st.cur;
  st.cur = start + s.tile1;
  return true;
}

__device__ __forceinline__ float* score_row(const TreeParams& p, const Segment& s, int r) {
  return p.scores + (((int64_t)s.b * p.kv_heads + s.h) * p.rows + r) * p.score_stride;
}

// Where a segment's result goes.
template <int D, int kRows>
struct Parts {
  static constexpr int kFloats = kRows * (D + 2);  // [rows] m, [rows] l, [rows][D] o
  // A CTA's first segment leaves part 0, a later one (its last) part 1.
  __device__ __forceinline__ static float* mine(const TreeParams& p, const Stretch& st) {
    return p.parts + (int64_t)(2 * blockIdx.x + (st.seg.begin == st.lo ? 0 : 1)) * kFloats;
  }
  // Part c of the item; its first CTA may have begun it behind another item.
  __device__ __forceinline__ static const float* of(const TreeParams& p, const Stretch& st, int c) {
    const Segment& s = st.seg;
    const int start = s.begin - s.tile0;
    const int second = c == 0 && start != s.first_cta * st.per ? 1 : 0;
    return p.parts + (int64_t)(2 * (s.first_cta + c) + second) * kFloats;
  }
};

// Four elements of an output row from its unnormalised sum, and (with weights)
// the row's log-sum-exp. Empty rows give zeros.
template <int kRows, typename T>
__device__ __forceinline__ void write_row(const TreeParams& p, const Segment& s,
                                          const unsigned long long* masks, int r, int e, float m,
                                          float l, float4 o) {
  const int row = s.mblock * kRows + r;
  if (row >= p.rows) return;
  const bool empty = masks[r] == 0;
  if (p.weights && e == 0)
    p.lse[((int64_t)s.b * p.kv_heads + s.h) * p.rows + row] = empty ? INFINITY : m + log2f(l);
  const float f = 1.f / l;
  o = empty ? make_float4(0.f, 0.f, 0.f, 0.f)
            : make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
  T* out = static_cast<T*>(p.out) + s.b * p.o_sb + (row / p.group) * p.o_sn +
           (s.h * p.group + row % p.group) * p.o_sh + e;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(out) = o;
  } else {
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(o.x, o.y), __floats2bfloat162_rn(o.z, o.w)};
    *reinterpret_cast<uint2*>(out) = *reinterpret_cast<uint2*>(h);
  }
}

// Merges rows row0 .. row0 + kCount - 1 of the item's parts, in the order of the
// tile list, and writes them out; kThreads threads call it, after the last
// ticket of the rows has been taken. A thread's elements of a part are loaded
// together, so that a part costs one latency.
template <int D, int kRows, int kCount, int kThreads, typename T>
__device__ __forceinline__ void merge_parts(const TreeParams& p, const Stretch& st,
                                            const unsigned long long* masks, int row0, int tid) {
  constexpr int kPieces = D / 4;
  constexpr int kMine = kCount * kPieces / kThreads;
  static_assert(kCount * kPieces % kThreads == 0, "the rows are shared out evenly");
  const Segment& s = st.seg;
  const int ctas = s.last_cta - s.first_cta + 1;
  float m[kMine], l[kMine];
  float4 o[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll 2
  for (int c = 0; c < ctas; ++c) {
    const float* x = Parts<D, kRows>::of(p, st, c);
    float m2[kMine], l2[kMine];
    float4 y[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int at = tid + i * kThreads, r = row0 + at / kPieces, e = at % kPieces * 4;
      m2[i] = __ldcg(x + r);
      l2[i] = __ldcg(x + kRows + r);
      y[i] = __ldcg(reinterpret_cast<const float4*>(x + 2 * kRows + r * D + e));
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const float now = fmaxf(m[i], m2[i]), ref = now == -INFINITY ? 0.f : now;
      const float a = fast_exp2(m[i] - ref), b = fast_exp2(m2[i] - ref);
      m[i] = now;
      l[i] = l[i] * a + l2[i] * b;
      o[i].x = o[i].x * a + y[i].x * b, o[i].y = o[i].y * a + y[i].y * b;
      o[i].z = o[i].z * a + y[i].z * b, o[i].w = o[i].w * a + y[i].w * b;
    }
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = tid + i * kThreads;
    write_row<kRows, T>(p, s, masks, row0 + at / kPieces, at % kPieces * 4, m[i], l[i], o[i]);
  }
}

// Takes a ticket of the item (one thread, once its CTA's part is in memory):
// true for the last of the item's CTAs, which also re-arms the counter.
__device__ __forceinline__ bool take_ticket(const Segment& s, int* counter) {
  const bool last = atomicAdd(counter, 1) == s.last_cta - s.first_cta;
  if (last) *counter = 0;
  return last;
}

// Byte offset of 16-byte piece `piece` of row `row` in a tile of `rows` rows of
// D bf16, as a 128-byte-swizzled TMA box lays it out: columns in blocks of 64
// elements, pieces permuted within a row's 128 bytes.
template <int D>
__device__ __forceinline__ int tile_at(int rows, int row, int piece) {
  return (piece >> 3) * rows * 128 + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}

// tree_prepare.cu: the query blocks, and the nodes' keys and values in the
// cache. `split`: q times the scale, in two bf16 parts.
int launch_prepare(int dtype, int head_dim, int block_rows, const TreeParams& p,
                   cudaStream_t stream);
// tree_attention_mma.cu: bf16, blocks of 16, 32 or 64 query rows.
int mma_ctas_per_sm(int head_dim, int block_rows);
int launch_mma(int head_dim, int block_rows, const TreeParams& p, cudaStream_t stream);

}  // namespace tree
}  // namespace asrback
