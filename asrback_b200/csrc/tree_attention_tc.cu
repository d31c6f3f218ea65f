// Draft-tree attention in bf16 on the 5th-generation tensor cores, sm_100a. The
// split of the work is tree_attention.cu's.
//
// A block of query rows (the nodes of a row times the query heads of one
// key/value head, up to 128) is one 128-row tcgen05 tile against the row's keys
// in tiles of 64. The call is bound by streaming the cache, so the TMA warps run
// ahead of everything through the CTA's whole stretch, across items. A segment's
// tiles are taken in pairs, whose scores are one product of 128 columns (in
// shared memory one of 64 reads the queries as long, for half the result); the
// softmax of each tile of a pair has warps of its own, which share the rows'
// references. The scores of the next pair are computed as soon as a pair's are
// in registers, beside its softmax and the products with the values of the pair
// before; an item's end is read by warps of its own, from one of two output
// accumulators, while the next item is under way. Roles:
//   warp 0      TMA: a segment's query block, the pairs' keys;
//   warp 2      TMA: the tiles' values. (Two warps, since one issues tiles more
//               slowly than they arrive.) A full pair or tile is one copy, of
//               others only the blocks of 16 positions that hold keys;
//   warp 1      TMEM allocation, S = Q K^T. A rotated query is two bf16 parts
//               (their sum has 2^-17 of rounding), whose products are added up
//               in S;
//   warp 3      O (+)= P V, and of the values behind the cached keys: zeros
//               behind the last node, nothing infinite or NaN. (Two warps issue
//               MMAs, since the waits and descriptors of a tile take one of them
//               longer than the tile's share of the stream.)
//   warps 4-7   softmax of a pair's first tile, warps 8-11 of its second: thread =
//               TMEM lane = query row; only the warps that hold rows run. A row's
//               reference moves, and its O is rescaled, only when a score passes
//               it by more than 8 (base 2);
//   warps 12-15 an item's end: output or part.
//
// Bound: HBM's stream, with the tensor pipe close behind: a pair of 64 KB takes
// 1480 ns of a GPU's share of it, its products 1530 cycles (16 of 128 x 128 x 16
// for the scores in two parts, 8 for the output), whose operands keep shared
// memory's port busy, so that a spilled register costs more than an exponential.
// Measured, with the preparation before and the merge behind: 8 rows x 64 nodes
// of up to 8192 keys, 8 heads of 128 (175 MB) 48 us, of which this kernel's 33 are
// 5.3 TB/s; 64 rows x 16 nodes of up to 1024 keys (183 MB) 51.5 us. Steps on the
// way for the two: scores of 64 columns and an accumulator per tile of a pair 61
// and 63 us; one per pair, few spills (16 to 20 bytes of a thread's are left; 112 to
// 144 took 53.7 and 60) 48.6 and 53; an item's fixed cost in the split
// 48 and 51.5. No gain: exponentials on the FMA pipe (49 and 55), blocks of up to
// 64 rows laid out twice, for the softmax to use more schedulers (53.5 for the
// second), other ring lengths.
#include <algorithm>

#include "tree_tma.cuh"

namespace asrback {
namespace {

using namespace tree;

constexpr int kThreads = 512;
constexpr int kPair = 2 * kTile;  // keys whose scores are one product
constexpr int kMaxUnits = 16;     // pairs of keys, and tiles of values, in their rings
constexpr float kMoveThreshold = 8.0f;
// TMEM: a pair's S, two buffers of a pair's P, two O, so that a segment's products
// begin while the last one's output is read.
constexpr int kTmemCols = 512;
constexpr int kColP = kPair;
constexpr int kColO = kColP + kPair;

// What a softmax warp hands to the item's end, per tile of the pairs and row.
struct RowState {
  float m, l;
  unsigned long long mask;
};

// Shared memory: the query blocks, the rings of keys and of values, then the
// rest. The tensor core reads 128 rows from a block's start whatever its rows:
// what follows are keys, as rows of no one.
struct Layout {
  int slots, slot_bytes, pairs, tiles, tile_bytes;  // rings: pairs of keys, tiles of values
  __host__ __device__ int keys() const { return slots * slot_bytes; }
  __host__ __device__ int values() const { return keys() + pairs * 2 * tile_bytes; }
  __host__ __device__ int rest() const { return values() + tiles * tile_bytes; }
};

constexpr int kOffStates = 0;                                // [tile of a pair][128] RowState
constexpr int kOffTops = kOffStates + 2 * 128 * 16;          // [tile of a pair][128] float
constexpr int kOffBars = kOffTops + 2 * 128 * 4;
// full, empty per unit of keys and of values; q_full, q_empty per block; s_full,
// s_free; p_full per P buffer and tile; p_free per P buffer; state_full,
// state_empty per tile of a pair; o_final, o_free per O
constexpr int kNumBars = 4 * kMaxUnits + 4 + 2 + 4 + 2 + 4 + 4;
constexpr int kOffInts = kOffBars + kNumBars * 8;            // scratch[16], odd_segment, tmem
constexpr int kOffList = (kOffInts + 20 * 4 + 15) / 16 * 16;
constexpr int kRead = 32;  // output columns that an item's end reads at a time
constexpr int rest_bytes(int batch) { return kOffList + list_bytes(batch); }
constexpr int kBudget = 227 * 1024 - 1024;  // less the alignment of the base

// Two floats in one operation.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long x, y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(x), "l"(y));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(x));
  return a;
}

// Eight columns of this thread's TMEM lane, multiplied by `a`.
__device__ __forceinline__ void scale8(uint32_t at, float a) {
  float v[8];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7])
      : "r"(at)
      : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= a;
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
      : "memory");
}

// Whether a predicate holds in any of the 64 threads that meet at barrier `id`.
__device__ __forceinline__ bool any_of_64(int id, bool x) {
  int any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 64, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<int>(x)), "r"(id)
      : "memory");
  return any != 0;
}

template <int D, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    tree_tc_kernel(const __grid_constant__ Maps maps, const __grid_constant__ TreeParams p,
                   const Layout lay) {
  using T = __nv_bfloat16;
  constexpr int kUnitBytes = kTile * D * 2;
  constexpr int kHalves = D / 64;  // 128-byte column blocks
  constexpr int kParts = kSplit ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* rest = smem + lay.rest();
  RowState* states = reinterpret_cast<RowState*>(rest + kOffStates);
  float* tops = reinterpret_cast<float*>(rest + kOffTops);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(rest + kOffBars);  // [unit]
  uint64_t* k_empty = k_full + kMaxUnits;
  uint64_t* v_full = k_empty + kMaxUnits;
  uint64_t* v_empty = v_full + kMaxUnits;
  uint64_t* q_full = v_empty + kMaxUnits;  // [block buffer]
  uint64_t* q_empty = q_full + 2;
  uint64_t* s_full = q_empty + 2;
  uint64_t* s_free = s_full + 1;
  uint64_t* p_full = s_free + 1;  // [P buffer][tile]
  uint64_t* p_free = p_full + 4;  // [P buffer]: its products are done
  uint64_t* state_full = p_free + 2;  // [tile of a pair] from here
  uint64_t* state_empty = state_full + 2;
  uint64_t* o_final = state_empty + 2;  // [O] from here
  uint64_t* o_free = o_final + 2;
  int* scratch = reinterpret_cast<int*>(rest + kOffInts);  // [16]
  int* odd_segment = scratch + 16;  // [O] the segment's nodes hold infinite or NaN values
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(odd_segment + 2);
  TileList list(rest + kOffList, p.batch);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row_warps = p.block_rows / 32;
  // Of a query buffer: the rows, then their masks and the nodes' flags.
  const int rows_bytes = kParts * kHalves * p.block_rows * 128;

  if (threadIdx.x == 0) {
    for (int u = 0; u < kMaxUnits; ++u) {
      mbar_init(&k_full[u], 1);
      mbar_init(&k_empty[u], 1);
      mbar_init(&v_full[u], 1);
      mbar_init(&v_empty[u], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      // The MMA warps and the softmax warps.
      mbar_init(&q_empty[s], 2 + 2 * row_warps);
      mbar_init(&p_full[s], row_warps);
      mbar_init(&p_full[2 + s], row_warps);
      mbar_init(&p_free[s], 1);
      mbar_init(&state_full[s], row_warps);
      mbar_init(&state_empty[s], row_warps);
      mbar_init(&o_final[s], 1);
      mbar_init(&o_free[s], row_warps);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, 2 * row_warps);
    fence_barrier_init();
  }
  if (warp == 1) tc::tmem_alloc(tmem_slot, kTmemCols);
  griddep_launch_dependents();
  tc::tc_fence_before();
  // The lengths and counts are older than the preparation kernel, which began
  // behind them: only what that kernel writes is waited for, further down.
  Stretch st = begin_stretch<kThreads>(p, list, scratch);  // has barriers: inits are visible
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Segment& sg = st.seg;
  auto wait = [](uint64_t* bar, int parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity & 1)) != 0;
  };
  // Between the softmax and the products, where a suspended waiter wakes late.
  auto spin = [](uint64_t* bar, int parity) {
    return __all_sync(0xffffffffu, mbar_spin_bounded(bar, parity & 1)) != 0;
  };
  auto tiles_of = [](const Segment& s) {
    return s.length + s.count > 0 ? s.tile1 - s.tile0 : 0;  // a skipped row has none
  };
  bool ok = true;
  // The same in every lane, and known to be: descriptors built from it are kept in
  // uniform registers, which the issue of an MMA reads.
  auto uniform = [](uint32_t x) { return __reduce_max_sync(0xffffffffu, x); };

  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------------- TMA
    const int which = warp >> 1;  // keys or values
    const int units = which ? lay.tiles : lay.pairs, step = which ? kTile : kPair;
    uint64_t* full = which ? v_full : k_full;
    uint64_t* empty = which ? v_empty : k_empty;
    uint8_t* ring = smem + (which ? lay.values() : lay.keys());
    const bool leader = tc::elect_one();
    if (leader) {
      tc::prefetch_tensormap(&maps.tile[which]);
      tc::prefetch_tensormap(&maps.tail[which]);
    }
    __syncwarp();
    const uint64_t policy = l2_evict_first_policy();
    bool waited = false;
    int loads = 0;  // of query blocks
    Turn unit, block;
    for (; ok && next_segment(p, list, st); block.next(lay.slots)) {
      // The query block is loaded as soon as its buffer is free, and at the
      // latest when the products could not go on without it: before the ring
      // waits for a unit that this segment itself has filled.
      const int slot = block.at, q_lap = block.lap;
      bool q_due = which == 0;
      auto load_q = [&](bool now) {
        if (!q_due || (!now && !waited)) return;
        if (!waited) griddep_wait();
        waited = true;
        if (q_lap > 0) {
          if (!now && !__all_sync(0xffffffffu, mbar_test(&q_empty[slot], (q_lap - 1) & 1))) return;
          ok = wait(&q_empty[slot], q_lap - 1);
        }
        q_due = false;
        if (ok) ++loads;
        if (ok && leader) {
          mbar_arrive_expect_tx(&q_full[slot], p.q_block_bytes);
          bulk_g2s(smem + slot * lay.slot_bytes, p.q_blocks + (int64_t)sg.item * p.q_block_bytes,
                   p.q_block_bytes, &q_full[slot], policy);
        }
        __syncwarp();
      };
      const int begin = sg.tile0 * kTile;
      const int end = min(begin + tiles_of(sg) * kTile, sg.length + sg.count);
      for (int i = 0, key = begin; key < end && ok; ++i, key += step) {
        load_q(i >= units);
        // What has nodes in it comes after the preparation.
        if (!waited && min(key + step, end) > sg.length) {
          load_q(true);
          if (!waited) griddep_wait();
          waited = true;
        }
        if (ok && unit.lap > 0) ok = wait(&empty[unit.at], unit.lap - 1);
        if (ok && leader) {
          uint8_t* to = ring + unit.at * step * D * 2;
          if (which)
            load_tile<D>(to, maps, 1, key, end - key, sg.h, sg.b, &full[unit.at]);
          else
            load_tile<D, kPair>(to, maps, 0, key, end - key, sg.h, sg.b, &full[unit.at]);
        }
        __syncwarp();
        if (ok) unit.next(units);
      }
      if (ok) load_q(true);
    }
    // A wait gave up: the copies in flight still have to land before the CTA
    // may end.
    if (!ok) {
      for (int u = 0; u < units; ++u) {
        const int laps = unit.lap + (u < unit.at ? 1 : 0);
        if (laps > 0) wait(&full[u], laps - 1);
      }
      for (int s = 0; s < lay.slots; ++s) {
        const int laps = (loads + lay.slots - 1 - s) / lay.slots;
        if (laps > 0) wait(&q_full[s], laps - 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ S = Q K^T
    const bool leader = tc::elect_one();
    const uint64_t q_desc = tc::sw128_desc(smem_addr(smem), 16, 1024);
    const uint64_t k_desc = tc::sw128_desc(smem_addr(smem + lay.keys()), 16, 1024);
    const uint32_t half_step = p.block_rows * 128 >> 4;
    Turn unit, block;
    int pair = 0;
    for (; ok && next_segment(p, list, st); block.next(lay.slots)) {
      const int tiles = tiles_of(sg), slot = block.at;
      ok = wait(&q_full[slot], block.lap);
      if (tiles == 0 && leader) mbar_arrive(&q_empty[slot]);
      for (int i = 0; i < tiles && ok; i += 2, unit.next(lay.pairs), ++pair) {
        const int u = unit.at;
        ok = wait(&k_full[u], unit.lap);
        if (pair > 0) ok = ok && spin(s_free, pair - 1);
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t t_s = uniform(tmem);
        const uint64_t qd = q_desc + uniform(slot * lay.slot_bytes >> 4);
        const uint64_t kd = k_desc + uniform(u * (kPair * D * 2 >> 4));
        const uint32_t idesc = uniform(i + 1 < tiles ? tc::idesc_bf16(128, kPair, false)
                                                     : tc::idesc_bf16(128, kTile, false));
        if (leader) {
#pragma unroll
          for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int c = 0; c < kHalves; ++c)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                tc::mma_ss(t_s, qd + (part * kHalves + c) * half_step + 2 * k,
                           kd + c * (kPair * 128 >> 4) + 2 * k, idesc,
                           part > 0 || c > 0 || k > 0);
          tc::mma_commit(s_full);
          tc::mma_commit(&k_empty[u]);
          if (i + 2 >= tiles) tc::mma_commit(&q_empty[slot]);
        }
        __syncwarp();
      }
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------- O (+)= P V
    const bool leader = tc::elect_one();
    constexpr uint32_t kIdesc = tc::idesc_bf16(128, D, true);
    const uint64_t v_desc = tc::sw128_desc(smem_addr(smem + lay.values()), kTile * 128, 1024);
    Turn unit, block, out, buffer;
    for (; ok && next_segment(p, list, st); block.next(lay.slots), out.next(2)) {
      const int tiles = tiles_of(sg), total = sg.length + sg.count;
      // The block ends with a flag per node: its value holds infinities or NaN.
      ok = wait(&q_full[block.at], block.lap);
      const uint8_t* flags = smem + block.at * lay.slot_bytes + rows_bytes + 8 * p.block_rows;
      const bool odd = __any_sync(0xffffffffu, ok && ((lane < sg.count && flags[lane]) ||
                                                      (lane + 32 < sg.count && flags[lane + 32])));
      if (lane == 0) mbar_arrive(&q_empty[block.at]);
      for (int i = 0; i < tiles && ok; ++i, unit.next(lay.tiles)) {
        const int x = i & 1, u = unit.at, s = buffer.at, key = (sg.tile0 + i) * kTile;
        const bool last = i == tiles - 1;
        ok = wait(&v_full[u], unit.lap);
        if (!ok) break;
        if (key + kTile > sg.length) {
          uint8_t* values = smem + lay.values() + u * kUnitBytes;
          const int nodes_end = min(total - key, kTile), rows_end = min((nodes_end + 15) & ~15, kTile);
          // Behind the last node: zeros, for the product with zero
          // probabilities.
          for (int at = nodes_end * (D / 8) + lane; at < rows_end * (D / 8); at += 32)
            *reinterpret_cast<uint4*>(values + tile_at(kTile, at / (D / 8), at % (D / 8))) =
                make_uint4(0u, 0u, 0u, 0u);
          // An infinite or NaN value becomes zero too, since that product
          // would pass it on to the nodes that do not see it: the item's end
          // adds it where it is seen.
          if (odd) {
            const int row0 = max(sg.length - key, 0);
            for (int at = row0 * (D / 8) + lane; at < nodes_end * (D / 8); at += 32) {
              uint4* to = reinterpret_cast<uint4*>(values +
                                                   tile_at(kTile, at / (D / 8), at % (D / 8)));
              uint4 v = *to;
              uint32_t* words = &v.x;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if ((words[j] & 0x7f80u) == 0x7f80u) words[j] &= 0xffff0000u;
                if ((words[j] & 0x7f800000u) == 0x7f800000u) words[j] &= 0xffffu;
              }
              *to = v;
            }
          }
          tc::fence_proxy_async();
          __syncwarp();
        }
        // The segment's first products overwrite an accumulator whose last
        // segment has been read.
        if (i == 0 && out.lap > 0) ok = wait(&o_free[out.at], out.lap - 1);
        ok = ok && spin(&p_full[2 * s + x], buffer.lap);
        // The second tile's softmax takes its turn in a pair of one tile too.
        if (last && x == 0) ok = ok && wait(&p_full[2 * s + 1], buffer.lap);
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t t_o = tmem + kColO + uniform(out.at) * D;
        const uint32_t t_p = tmem + kColP + uniform(2 * s + x) * (kTile / 2);
        const uint64_t vd = v_desc + uniform(u * (kUnitBytes >> 4));
        if (leader) {
          if (i == 0) {
            odd_segment[out.at] = odd;
            __threadfence_block();
          }
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k)
            if (16 * k < total - key)
              tc::mma_ts(t_o, t_p + 8 * k, vd + (k * 2048 >> 4), kIdesc, i > 0 || k > 0);
          if (last) tc::mma_commit(&o_final[out.at]);
          if (last || x == 1) tc::mma_commit(&p_free[s]);
          tc::mma_commit(&v_empty[u]);
        }
        __syncwarp();
        if (last || x == 1) buffer.next(2);
      }
      // A segment without tiles takes its turn all the same: two phases of a
      // barrier in a row would look alike.
      if (tiles == 0) {
        if (out.lap > 0) ok = ok && wait(&o_free[out.at], out.lap - 1);
        if (leader) mbar_arrive(&o_final[out.at]);
      }
    }
  } else if (warp >= 4 && warp < 12 && (warp & 3) < row_warps) {
    // --------------------------------------------------------------- softmax
    const int x = (warp >> 2) - 1, quarter = warp & 3;
    const int r = 32 * quarter + lane;  // this thread's row of the block
    const uint32_t lanes = static_cast<uint32_t>(32 * quarter) << 16;
    Turn block, out, buffer;
    int pair = 0;
    for (int n = 0; next_segment(p, list, st); ++n, block.next(lay.slots), out.next(2)) {
      const int slot = block.at;
      if (ok) ok = wait(&q_full[slot], block.lap);
      const unsigned long long mask =
          ok ? reinterpret_cast<const unsigned long long*>(smem + slot * lay.slot_bytes +
                                                           rows_bytes)[r]
             : 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[slot]);
      float m = -INFINITY, l = 0.f;  // m: the same for both tiles of a pair
      const int tiles = tiles_of(sg);
      // A wait that gives up ends the work, but not the turns at the barriers that
      // the two tiles' warps share.
      for (int i = 0; i < tiles; i += 2, ++pair, buffer.next(2)) {
        if (ok) ok = spin(s_full, pair);
        // The second tile of a pair of one takes part in all but the work.
        const bool here = ok && i + x < tiles;
        float s[kTile];
        float highest = -INFINITY;
        if (here) {
          tc::tc_fence_after();
          tc::tmem_ld64(tmem + lanes + x * kTile, s);
          tc::tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        if (here) {
          if constexpr (!kSplit) {
#pragma unroll
            for (int j = 0; j < kTile; ++j) s[j] *= p.scale_log2;
          }
          const int cached = sg.length - (sg.tile0 + i + x) * kTile;  // columns before the nodes
          if (cached < kTile) {
            // Behind the cached keys lie the nodes, behind them nothing (a mask
            // has no bits there).
            const unsigned long long older = cached > 0 ? (1ull << cached) - 1 : 0;
            const unsigned long long seen =
                older | (cached >= 0 ? mask << cached : mask >> -cached);
#pragma unroll
            for (int j = 0; j < kTile; ++j)
              if ((seen >> j & 1) == 0) s[j] = -INFINITY;
          }
          float top[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) top[j] = fmaxf(s[j], s[j + 4]);
#pragma unroll
          for (int j = 8; j < kTile; j += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) top[k] = fmax3(top[k], s[j + k], s[j + k + 4]);
          highest = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        }
        // Both tiles' warps of the rows agree on the references.
        if (any_of_64(2 + quarter, highest > m + kMoveThreshold)) {
          tops[128 * x + r] = highest;
          any_of_64(2 + quarter, false);
          const float top = fmaxf(highest, tops[128 * (1 - x) + r]);
          const float now = top > m + kMoveThreshold ? top : m;
          const float a = now == m ? 1.f : fast_exp2(m - now);
          if (i > 0 && x == 0) {
            // The segment's O has to be at rest: its last pair's products are done.
            const Turn before = buffer.at ? Turn{0, buffer.lap} : Turn{1, buffer.lap - 1};
            if (ok) ok = wait(&p_free[before.at], before.lap);
            tc::tc_fence_after();
            const uint32_t t_o = tmem + lanes + kColO + out.at * D;
#pragma unroll
            for (int c = 0; c < D; c += 8) scale8(t_o + c, a);
            tc::tmem_wait_st();
          }
          l *= a;
          m = now;
        }
        // The buffer's products of two pairs before are done.
        if (buffer.lap > 0) ok = ok && spin(&p_free[buffer.at], buffer.lap - 1);
        if (here) {
          // Probabilities are rounded to bf16 for the second product (2^-8 at
          // most, against an output in bf16 itself); their sum is not.
          const float ref = m == -INFINITY ? 0.f : m;
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          const uint32_t t_p = tmem + lanes + kColP + (2 * buffer.at + x) * (kTile / 2);
#pragma unroll
          for (int part = 0; part < kTile; part += 32) {
            uint32_t packed[16];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float2 e = add2(make_float2(s[part + j], s[part + j + 1]), make_float2(-ref, -ref));
              e = make_float2(fast_exp2(e.x), fast_exp2(e.y));
              sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], e);
              packed[j / 2] = tc::bf16x2(e.x, e.y);
            }
            tc::tmem_st16(t_p + part / 2, packed);
          }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          tc::tmem_wait_st();
          tc::tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * buffer.at + x]);
      }
      if (n > 0 && ok) ok = wait(&state_empty[x], n - 1);
      states[128 * x + r] = RowState{m, l, mask};
      __syncwarp();
      if (lane == 0) mbar_arrive(&state_full[x]);
    }
  } else if (warp >= 12 && (warp & 3) < row_warps) {
    // ---------------------------------------------------------- an item's end
    const int quarter = warp & 3, r = 32 * quarter + lane;
    const uint32_t lanes = static_cast<uint32_t>(32 * quarter) << 16;
    Turn from;
    for (int n = 0; next_segment(p, list, st); ++n, from.next(2)) {
      const uint32_t t_o = tmem + lanes + kColO + from.at * D;
      const int tiles = tiles_of(sg);
      const bool whole = sg.whole();
      const int row = sg.mblock * p.block_rows + r;
      float* part = Parts<D>::mine(p, st);
      ok = ok && wait(&state_full[0], n) && wait(&state_full[1], n);
      const RowState a = states[r], b = states[128 + r];
      const float m = a.m, l = a.l + b.l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&state_empty[0]), mbar_arrive(&state_empty[1]);
      ok = ok && wait(&o_final[from.at], from.lap);
      tc::tc_fence_after();
      const bool odd = tiles > 0 && odd_segment[from.at] != 0;
      const bool live = row < p.rows;
      const float f = whole ? 1.f / l : 1.f;
      T* out = out_row<T>(p, sg.b, sg.h, live ? row : 0);
#pragma unroll
      for (int c = 0; c < D; c += kRead) {
        float o[kRead];
        tc::tmem_ld32(t_o + c, o);
        if (c == D - kRead) {
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_free[from.at]);
        }
#pragma unroll
        for (int i = 0; i < kRead; ++i) o[i] = tiles > 0 ? o[i] * f : 0.f;
        if (odd) {
          // The infinite and NaN values of the nodes that the row sees, among
          // the segment's tiles.
          for (int i = 0; i < sg.count; ++i) {
            const int at = sg.length + i - sg.tile0 * kTile;
            if ((a.mask >> i & 1) == 0 || at < 0 || at >= tiles * kTile) continue;
            const T* v = static_cast<const T*>(p.value_cache) + sg.b * p.c_sb +
                         (int64_t)(sg.length + i) * p.c_sp + sg.h * p.c_sh + c;
#pragma unroll
            for (int j = 0; j < kRead; ++j) {
              const float value = __bfloat162float(v[j]);
              if (!(fabsf(value) < INFINITY)) o[j] += value;
            }
          }
        }
        if (!live) continue;
        if (whole) {
          uint32_t w[kRead / 2];
#pragma unroll
          for (int i = 0; i < kRead / 2; ++i)
            w[i] = a.mask == 0 ? 0u : tc::bf16x2(o[2 * i], o[2 * i + 1]);
#pragma unroll
          for (int i = 0; i < kRead / 2; i += 4)
            *reinterpret_cast<uint4*>(out + c + 2 * i) =
                make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < kRead; i += 4)
            *reinterpret_cast<float4*>(part + Parts<D>::at(p, r, c + i)) =
                make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
      if (live && !whole) part[r] = m, part[p.block_rows + r] = l;
    }
  }
  if (!ok && lane == 0 && p.status) atomicOr(p.status, ASRBACK_STATUS_TIMEOUT);
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

template <int D, bool kSplit>
int launch(const TreeParams& p, cudaStream_t stream) {
  auto kernel = tree_tc_kernel<D, kSplit>;
  Maps maps;
  if (int rc = make_maps(&maps, p, D, kPair)) return rc;
  static thread_local int prepared_device = -1;
  int device = 0;
  if (int rc = check_cuda(cudaGetDevice(&device), "cudaGetDevice")) return rc;
  if (prepared_device != device) {
    if (int rc = check_cuda(cudaFuncSetAttribute(
                                kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024),
                            "cudaFuncSetAttribute(tree attention)"))
      return rc;
    prepared_device = device;
  }
  // Two query blocks where they leave the ring most of the shared memory.
  Layout lay{};
  lay.slot_bytes = (p.q_block_bytes + 1023) / 1024 * 1024;
  lay.slots = lay.slot_bytes <= 40 * 1024 ? 2 : 1;
  lay.tile_bytes = kTile * D * 2;
  // At least eight tiles' room: half of it, or the lesser part, for the keys.
  const int room = (kBudget - rest_bytes(p.batch) - lay.keys()) / lay.tile_bytes;
  lay.pairs = (room + 1) / 4;
  lay.tiles = std::min(room - 2 * lay.pairs, kMaxUnits);
  return launch_pdl(kernel, dim3(p.ctas), dim3(kThreads), 1024 + lay.rest() + rest_bytes(p.batch),
                    stream, "tree attention launch", maps, p, lay);
}

}  // namespace

namespace tree {

int launch_tc(int head_dim, const TreeParams& p, cudaStream_t stream) {
  if (head_dim == 64) return p.q_norm ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
  return p.q_norm ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
}

}  // namespace tree
}  // namespace asrback
