// What the draft-tree attention kernels share: the stretch of the tile list
// that a CTA works through, the query rows' and the tree's own tile's
// preparation, and the end of a segment (output, or part and merge).
#pragma once

#include "common.cuh"

namespace asrback {
namespace tree {

constexpr int kTile = 64;            // keys per tile; the tree (at most 64 nodes) is one tile
constexpr int kThreads = 128;
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
  int* counters;  // one per item, zero between calls
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

__device__ __forceinline__ int row_tiles(int length) { return (length + kTile - 1) / kTile + 1; }

template <int kRows>
struct Common {
  unsigned long long mask[kRows];  // the tree's nodes that a query row sees; 0: an empty row
  int prefix[kMaxBatch];           // tiles of rows 0..b
  uint32_t span[kMaxBatch];        // length << 7 | count
  int warp_sum[kThreads / 32];
  int is_last;
};

struct Segment {
  int b, h, mblock, item;
  int length, count;
  int tiles;         // of the item: cache tiles, then the tree
  int tile0, tile1;  // this segment's
  int begin;         // tile0 in the list of all tiles
  int first_cta, last_cta;
  __device__ __forceinline__ int tile_keys(int first_key) const {
    return first_key == length ? count : length - first_key;
  }
};

// A CTA's stretch [lo, hi) of the list of all items' tiles, `per` tiles each.
struct Stretch {
  int lo, hi, cur, per, row;
  Segment seg;
};

template <int kRows>
__device__ __forceinline__ Stretch begin_stretch(const TreeParams& p, Common<kRows>& cm) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int carry = 0;
  for (int base = 0; base < p.batch; base += kThreads) {
    const int b = base + tid;
    int tiles = 0;
    if (b < p.batch) {
      const RowSpan s = row_span(p, b);
      if (s.bad && blockIdx.x == 0 && p.status) atomicOr(p.status, ASRBACK_STATUS_POSITION);
      cm.span[b] = static_cast<uint32_t>(s.length) << 7 | s.count;
      tiles = row_tiles(s.length) * p.kv_heads * p.mblocks;
    }
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) cm.warp_sum[warp] = sum;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) sum += cm.warp_sum[w];
    }
    if (b < p.batch) cm.prefix[b] = sum + carry;
    for (int w = 0; w < kThreads / 32; ++w) carry += cm.warp_sum[w];
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
    if (cm.prefix[mid] > st.lo) high = mid;
    else low = mid + 1;
  }
  st.row = low;
  return st;
}

// The next (part of an) item of the stretch; false at its end.
template <int kRows>
__device__ __forceinline__ bool next_segment(const TreeParams& p, const Common<kRows>& cm,
                                             Stretch& st) {
  if (st.cur >= st.hi) return false;
  while (cm.prefix[st.row] <= st.cur) ++st.row;
  Segment& s = st.seg;
  const int base = st.row > 0 ? cm.prefix[st.row - 1] : 0;
  s.b = st.row;
  s.length = static_cast<int>(cm.span[s.b] >> 7);
  s.count = static_cast<int>(cm.span[s.b] & 127u);
  s.tiles = row_tiles(s.length);
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

// A lane's D / 32 consecutive elements of a row.
template <int D, typename T>
__device__ __forceinline__ void load_lane(const void* row, int lane, float* x) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (D == 128) {
      const float4 v = __ldg(static_cast<const float4*>(row) + lane);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
      const float2 v = __ldg(static_cast<const float2*>(row) + lane);
      x[0] = v.x, x[1] = v.y;
    }
  } else {
    uint32_t u[D / 64];
    if constexpr (D == 128) {
      const uint2 v = __ldg(static_cast<const uint2*>(row) + lane);
      u[0] = v.x, u[1] = v.y;
    } else {
      u[0] = __ldg(static_cast<const uint32_t*>(row) + lane);
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
}

template <int D, typename T>
__device__ __forceinline__ void store_lane(void* row, int lane, const float* x) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (D == 128)
      static_cast<float4*>(row)[lane] = make_float4(x[0], x[1], x[2], x[3]);
    else
      static_cast<float2*>(row)[lane] = make_float2(x[0], x[1]);
  } else {
    __nv_bfloat162 h[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    if constexpr (D == 128)
      static_cast<uint2*>(row)[lane] = *reinterpret_cast<uint2*>(h);
    else
      static_cast<uint32_t*>(row)[lane] = *reinterpret_cast<uint32_t*>(h);
  }
}

// RMSNorm, then rotate-half rotary embedding of one head's row, D / 32
// consecutive elements per lane, all in float32: element d pairs with d +- D/2,
// which lane ^ 16 holds.
template <int D, typename T>
__device__ __forceinline__ void norm_rotate(const TreeParams& p, const void* weight, int64_t place,
                                            int lane, float* x) {
  constexpr int E = D / 32;
  float w[E], cs[E], sn[E];
  load_lane<D, T>(weight, lane, w);
  load_lane<D, T>(static_cast<const T*>(p.cos) + place * p.table_stride, lane, cs);
  load_lane<D, T>(static_cast<const T*>(p.sin) + place * p.table_stride, lane, sn);
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < E; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float r = rsqrtf(ss / D + p.eps);
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const float y = x[j] * r * w[j];
    const float pair = __shfl_xor_sync(0xffffffffu, y, 16);
    x[j] = y * cs[j] + (lane < 16 ? -pair : pair) * sn[j];
  }
}

// The block's query rows: row r is node r / group, head r % group. Fills
// cm.mask and calls store(row, element, values, count) for each lane's piece;
// empty rows (no such node, or a mask without bits) are zeros.
template <int D, int kRows, typename T, typename Store>
__device__ __forceinline__ void prepare_rows(const TreeParams& p, const Segment& s,
                                             Common<kRows>& cm, int warp, int lane, Store store) {
  constexpr int E = D / 32;
  const unsigned long long live = s.count >= 64 ? ~0ull : (1ull << s.count) - 1;
  const int64_t position = p.q_norm ? p.positions[s.b] : 0;
#pragma unroll 4
  for (int i = 0; i < kRows / 4; ++i) {
    const int r = warp + 4 * i, row = s.mblock * kRows + r;
    const int node = row / p.group, head = s.h * p.group + row % p.group;
    float x[E];
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = 0.f;
    unsigned long long mask = 0;
    if (row < p.rows && node < s.count) {
      mask = static_cast<unsigned long long>(__ldg(p.ancestors + (int64_t)s.b * p.nodes + node)) &
             live;
      if (mask) {
        load_lane<D, T>(static_cast<const T*>(p.q) + s.b * p.q_sb + node * p.q_sn + head * p.q_sh,
                        lane, x);
        if (p.q_norm) {
          const int depth = min(max(__ldg(p.depths + (int64_t)s.b * p.nodes + node), 0), node);
          norm_rotate<D, T>(p, p.q_norm, position + depth, lane, x);
        }
      }
    }
    if (lane == 0) cm.mask[r] = mask;
    store(r, lane * E, x, E);
  }
}

// The tree's keys and values: normalised and rotated, rounded to T, written to
// the cache (by the first block of query rows) and handed to store(node,
// element, key, value, count). Nodes up to the next multiple of 16 are zeros.
// Returns, after a barrier, whether every value is finite.
template <int D, typename T, int kRows, typename Store>
__device__ __forceinline__ bool load_tree_tile(const TreeParams& p, const Segment& s,
                                               Common<kRows>& cm, int warp, int lane, Store store) {
  constexpr int E = D / 32;
  const int64_t position = p.q_norm ? p.positions[s.b] : 0;
  bool finite = true;
#pragma unroll 2
  for (int i = warp; i < (s.count + 15) / 16 * 16; i += 4) {
    float k[E], v[E];
#pragma unroll
    for (int j = 0; j < E; ++j) k[j] = v[j] = 0.f;
    if (i < s.count) {
      load_lane<D, T>(static_cast<const T*>(p.k) + s.b * p.k_sb + i * p.k_sn + s.h * p.k_sh, lane,
                      k);
      load_lane<D, T>(static_cast<const T*>(p.v) + s.b * p.v_sb + i * p.v_sn + s.h * p.v_sh, lane,
                      v);
      if (p.q_norm) {
        const int depth = min(max(__ldg(p.depths + (int64_t)s.b * p.nodes + i), 0), i);
        norm_rotate<D, T>(p, p.k_norm, position + depth, lane, k);
      }
      if (s.mblock == 0) {
        const int64_t at = s.b * p.c_sb + (int64_t)(s.length + i) * p.c_sp + s.h * p.c_sh;
        store_lane<D, T>(static_cast<T*>(p.key_cache) + at, lane, k);
        store_lane<D, T>(static_cast<T*>(p.value_cache) + at, lane, v);
      }
#pragma unroll
      for (int j = 0; j < E; ++j) finite &= fabsf(v[j]) < INFINITY;
    }
    store(i, lane * E, k, v, E);
  }
  return __syncthreads_and(finite) != 0;
}

// The end of a segment. get(row, element, m, l, o) gives the CTA's state of a
// query row and four elements of its unnormalised output. An item that lies
// in one CTA is written out; otherwise the part goes to the workspace and the
// item's last CTA merges all of them, in the order of the tile list.
template <int D, int kRows, typename T, typename Get>
__device__ __forceinline__ void finish_segment(const TreeParams& p, const Stretch& st,
                                               Common<kRows>& cm, Get get) {
  constexpr int kPieces = D / 4;
  constexpr int kPart = kRows * (D + 2);
  const Segment& s = st.seg;
  const int tid = threadIdx.x;
  auto write = [&](int r, int e, float m, float l, float4 o) {
    const int row = s.mblock * kRows + r;
    if (row >= p.rows) return;
    const bool empty = cm.mask[r] == 0;
    if (p.weights && e == 0)
      p.lse[((int64_t)s.b * p.kv_heads + s.h) * p.rows + row] = empty ? INFINITY : m + log2f(l);
    const float f = empty ? 0.f : 1.f / l;
    if (empty) o = make_float4(0.f, 0.f, 0.f, 0.f);
    T* out = static_cast<T*>(p.out) + s.b * p.o_sb + (row / p.group) * p.o_sn +
             (s.h * p.group + row % p.group) * p.o_sh + e;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(out) = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
    } else {
      __nv_bfloat162 h[2] = {__floats2bfloat162_rn(o.x * f, o.y * f),
                             __floats2bfloat162_rn(o.z * f, o.w * f)};
      *reinterpret_cast<uint2*>(out) = *reinterpret_cast<uint2*>(h);
    }
  };
  if (s.first_cta == s.last_cta) {
    for (int i = tid; i < kRows * kPieces; i += kThreads) {
      float m, l;
      float4 o;
      get(i / kPieces, i % kPieces * 4, m, l, o);
      write(i / kPieces, i % kPieces * 4, m, l, o);
    }
    return;
  }
  // A CTA's first segment leaves part 0, a later one (its last) part 1.
  const int cta = blockIdx.x;
  float* part = p.parts + (int64_t)(2 * cta + (s.begin == st.lo ? 0 : 1)) * kPart;
  for (int i = tid; i < kRows * kPieces; i += kThreads) {
    const int r = i / kPieces, e = i % kPieces * 4;
    float m, l;
    float4 o;
    get(r, e, m, l, o);
    if (e == 0) part[r] = m, part[kRows + r] = l;
    *reinterpret_cast<float4*>(part + 2 * kRows + r * D + e) = o;
  }
  __threadfence();
  __syncthreads();
  const int ctas = s.last_cta - s.first_cta + 1;
  if (tid == 0) {
    cm.is_last = atomicAdd(p.counters + s.item, 1) == ctas - 1;
    if (cm.is_last) p.counters[s.item] = 0;
  }
  __syncthreads();
  if (!cm.is_last) return;
  __threadfence();
  // The item's first CTA may have begun it behind another item (part 1).
  const int start = s.begin - s.tile0;
  const float* parts0 =
      p.parts + (int64_t)(2 * s.first_cta + (start == s.first_cta * st.per ? 0 : 1)) * kPart;
  auto part_of = [&](int c) {
    return c == 0 ? parts0 : p.parts + (int64_t)(2 * (s.first_cta + c)) * kPart;
  };
  for (int i = tid; i < kRows * kPieces; i += kThreads) {
    const int r = i / kPieces, e = i % kPieces * 4;
    if (s.mblock * kRows + r >= p.rows) continue;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < ctas; ++c) m = fmaxf(m, __ldcg(part_of(c) + r));
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int c = 0; c < ctas; ++c) {
      const float* x = part_of(c);
      const float a = fast_exp2(__ldcg(x + r) - ref);
      const float4 y = __ldcg(reinterpret_cast<const float4*>(x + 2 * kRows + r * D + e));
      l = fmaf(__ldcg(x + kRows + r), a, l);
      o.x = fmaf(y.x, a, o.x), o.y = fmaf(y.y, a, o.y);
      o.z = fmaf(y.z, a, o.z), o.w = fmaf(y.w, a, o.w);
    }
    write(r, e, m, l, o);
  }
}

}  // namespace tree
}  // namespace asrback
