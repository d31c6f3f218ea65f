// Draft-tree attention in bf16 for up to 16 query rows per key/value head (nodes x
// heads / kv_heads), with head_dim 64 up to 32: mma.sync with a TMA warp, sm_100a.
// The split of the work is tree_attention.cu's.
//
// The call is bound by streaming the cache, so the TMA warp runs ahead of the
// products through the CTA's whole stretch, across items, and waits for nothing
// but a free ring unit (and once for the preparation kernel, which it overlaps
// with the first cached tiles). Roles:
//   warp 4    TMA: a segment's query block; a tile's keys, then its values, each
//             one ring unit of 64 positions x D (128-byte swizzle);
//   warps 0-3 the products. For the scores each warp takes 16 of a tile's 64
//             keys; the probabilities meet in shared memory, and for the output
//             each warp takes a quarter of the columns, over all keys: no merge
//             of outputs between warps, and a quarter of its registers.
// One barrier per tile among the four: the scores of tile t + 1 are computed
// before it, so that the barrier which publishes tile t's probabilities also
// votes on whether a row of tile t + 1 passes its softmax reference by more than
// 8 (base 2); only then the references move.
//
// mma.sync instead of tcgen05: 16 rows would leave seven eighths of a 128-row tcgen05
// tile empty, and its softmax to half of one warp. Four warps share it
// here, and their products issue as fast as the cache arrives (measured: one
// m16n8k16 in 2.05 cycles per SM). Bound: HBM's stream, for items of few tiles
// an item's fixed cost too. Measured, with the preparation before and the merge
// behind: 64 rows x 1 node of up to 1024 keys, 8 heads of 128, with weights (171
// MB) 45 us, of which this kernel's 32 are 5.3 TB/s; 3 rows x 4 nodes of up to
// 16384 keys, with weights (128 MB) 39 us; 64 rows x 8 nodes of up to 448 keys, 20
// heads of 64 (98 MB) 30 us, of which this kernel's 21 are 4.6 TB/s; 1 row x 6
// nodes of 256 keys 8.5 us. With head_dim 64 a second block of 16 rows shares the
// fragments of keys and values.
#include "tree_tma.cuh"

namespace asrback {
namespace {

using namespace tree;

constexpr int kWarps = 4;  // that compute
constexpr int kThreads = 32 * (kWarps + 1);
constexpr float kMoveThreshold = 8.0f;
constexpr int kMaxUnits = 16;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Barrier among the computing warps that tells all whether any thread voted.
__device__ __forceinline__ bool sync_any(bool vote) {
  uint32_t any;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %1, 0;\n"
      "barrier.cta.red.or.pred q, 1, 128, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(any)
      : "r"(vote ? 1u : 0u)
      : "memory");
  return any != 0;
}
__device__ __forceinline__ void sync_warps() { named_sync(1, 32 * kWarps); }

// CTAs per SM: as many as registers and shared memory allow, since a tile's
// chain of products, barrier and exponentials and an item's end are latencies
// that only other CTAs' work fills.
constexpr int ctas_per_sm(int head_dim, int rows) {
  return head_dim == 64 && rows == 16 ? 4 : 3;
}

// kBlocks: of 16 query rows.
template <int D, bool kSplit, int kBlocks>
struct Shape {
  static constexpr int kRows = 16 * kBlocks;
  static constexpr int kPerSm = ctas_per_sm(D, kRows);
  static constexpr int kUnitBytes = kTile * D * 2;  // keys or values of a tile
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kBlockBytes = (kSplit ? 2 : 1) * kQBytes + kRows * 8 + kMaxNodes;
  static constexpr int kSlotBytes = (kBlockBytes + 127) / 128 * 128;
  static constexpr int kQSlots = D == 64 ? 2 : 1;
  static constexpr int kOffP = kQSlots * kSlotBytes;  // [2][rows][64 keys]
  static constexpr int kPBytes = kRows * kTile * 2;
  static constexpr int kOffRing = (kOffP + 2 * kPBytes + 1023) / 1024 * 1024;
  // row_top, row_sum[2], scratch, barriers, then the tile list; slack to align
  // the base to 1024.
  static constexpr int kMisc = 3 * kWarps * kRows * 4 + 64 + (2 * kMaxUnits + 4) * 8;
  static constexpr int kBudget = (228 * 1024 / kPerSm - 1024) / 16 * 16;
  static constexpr int units(int batch) {
    const int n = (kBudget - 1024 - kOffRing - kMisc - list_bytes(batch)) / kUnitBytes;
    return n > kMaxUnits ? kMaxUnits : n;
  }
  static constexpr int bytes(int units, int batch) {
    return 1024 + kOffRing + units * kUnitBytes + kMisc + list_bytes(batch);
  }
  // A tile's keys are read before the last tile's values: three units make
  // progress.
  static_assert(units(kMaxBatch) >= 3, "the ring is too short");
};

template <int D, bool kSplit, int kBlocks, bool kWeights>
__global__ void __launch_bounds__(kThreads, Shape<D, kSplit, kBlocks>::kPerSm)
    tree_mma_kernel(const __grid_constant__ Maps maps, const __grid_constant__ TreeParams p,
                    const int units) {
  using Sh = Shape<D, kSplit, kBlocks>;
  using T = __nv_bfloat16;
  constexpr int kRows = Sh::kRows;
  constexpr int kQSlots = Sh::kQSlots;
  constexpr int kCols = D / kWarps;  // output columns of a warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* misc = smem + Sh::kOffRing + units * Sh::kUnitBytes;
  float* row_top = reinterpret_cast<float*>(misc);                       // [warp][rows]
  float* row_sums = row_top + kWarps * kRows;                            // [2][warp][rows]
  int* scratch = reinterpret_cast<int*>(row_sums + 2 * kWarps * kRows);  // [16]
  uint64_t* full = reinterpret_cast<uint64_t*>(scratch + 16);            // [unit]
  uint64_t* empty = full + kMaxUnits;
  uint64_t* q_full = empty + kMaxUnits;  // [slot]
  uint64_t* q_empty = q_full + kQSlots;
  TileList list(misc + Sh::kMisc, p.batch);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int u = 0; u < units; ++u) {
      mbar_init(&full[u], 1);
      mbar_init(&empty[u], kWarps);
    }
    for (int s = 0; s < kQSlots; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], kWarps);
    }
    fence_barrier_init();
  }
  griddep_launch_dependents();
  // The lengths and counts are older than the preparation kernel, which began
  // behind them: only what that kernel writes is waited for, further down.
  Stretch st = begin_stretch<kThreads>(p, list, scratch);  // has a barrier: inits are visible
  const Segment& sg = st.seg;
  auto wait = [](uint64_t* bar, int parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity & 1)) != 0;
  };
  bool ok = true;

  if (warp == kWarps) {
    // ------------------------------------------------------------------- TMA
    const bool leader = tc::elect_one();
    if (leader) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        tc::prefetch_tensormap(&maps.tile[i]);
        tc::prefetch_tensormap(&maps.tail[i]);
      }
    }
    __syncwarp();
    const uint64_t policy = l2_evict_first_policy();
    bool waited = false;
    int loads = 0;  // of query blocks
    Turn unit, block;
    for (; ok && next_segment(p, list, st); block.next(kQSlots)) {
      // The query block is loaded as soon as its buffer is free, and at the
      // latest when the products could not go on without it: before the ring
      // waits for a unit that this segment itself has filled.
      bool q_due = true;
      auto load_q = [&](bool now) {
        if (!q_due || (!now && !waited)) return;
        if (!waited) griddep_wait();
        waited = true;
        if (block.lap > 0) {
          uint64_t* bar = &q_empty[block.at];
          if (!now && !__all_sync(0xffffffffu, mbar_test(bar, (block.lap - 1) & 1))) return;
          ok = wait(bar, block.lap - 1);
        }
        q_due = false;
        if (ok) ++loads;
        if (ok && leader) {
          mbar_arrive_expect_tx(&q_full[block.at], Sh::kBlockBytes);
          bulk_g2s(smem + block.at * Sh::kSlotBytes,
                   p.q_blocks + (int64_t)sg.item * Sh::kBlockBytes, Sh::kBlockBytes,
                   &q_full[block.at], policy);
        }
        __syncwarp();
      };
      const int total = sg.length + sg.count;
      int filled = 0;  // units of this segment
      for (int tile = sg.tile0; tile < sg.tile1 && ok && total > 0; ++tile) {
        const int key = tile * kTile, keys = min(kTile, total - key);
        // A tile with nodes in it comes after the preparation.
        if (!waited && key + kTile > sg.length) load_q(true);
        for (int which = 0; which < 2 && ok; ++which, ++filled) {
          load_q(filled >= units);
          if (ok && unit.lap > 0) ok = wait(&empty[unit.at], unit.lap - 1);
          if (ok && leader)
            load_tile<D>(smem + Sh::kOffRing + unit.at * Sh::kUnitBytes, maps, which, key, keys,
                         sg.h, sg.b, &full[unit.at]);
          __syncwarp();
          if (ok) unit.next(units);
        }
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
      for (int s = 0; s < kQSlots; ++s) {
        const int laps = (loads + kQSlots - 1 - s) / kQSlots;
        if (laps > 0) wait(&q_full[s], laps - 1);
      }
    }
  } else {
    // -------------------------------------------------------------- products
    const int quad = lane & 3, row0 = lane >> 2;  // of each block rows row0 and row0 + 8
    const uint32_t base = smem_addr(smem);
    const uint32_t ring = base + Sh::kOffRing;
    // ldmatrix: lane l gives the address of row l % 8 of matrix l / 8. Tiles start
    // on 128-byte boundaries and rows are a multiple of eight apart, so a lane's
    // swizzle is its own: piece 2 k + j of its row lies at (row + (j ^ l % 8)
    // pieces) ^ 2 k pieces.
    const int mat = lane >> 3, mrow = lane & 7;
    const uint32_t k_lane = (16 * warp + (mat >> 1) * 8 + mrow) * 128 + (((mat & 1) ^ mrow) << 4);
    const uint32_t q_lane = ((mat & 1) * 8 + mrow) * 128 + (((mat >> 1) ^ mrow) << 4);
    uint32_t v_lane[kCols / 16];
#pragma unroll
    for (int c = 0; c < kCols / 16; ++c)
      v_lane[c] = tile_at(kTile, (mat & 1) * 8 + mrow, warp * (kCols / 8) + 2 * c + (mat >> 1));
    // Where the lane's probabilities go: rows row0, row0 + 8, two pieces each.
    const uint32_t p_store = row0 * 128 + (((2 * warp) ^ (row0 & 7)) << 4) + 4 * quad;
    Turn unit, block;
    int parity = 0;  // of the probabilities' buffer, through all tiles
    for (int n = 0; next_segment(p, list, st); ++n, block.next(kQSlots)) {
      const uint32_t q_at = base + block.at * Sh::kSlotBytes;
      const uint8_t* flags = smem + block.at * Sh::kSlotBytes + Sh::kBlockBytes - kMaxNodes;
      const auto* masks = reinterpret_cast<const unsigned long long*>(flags) - kRows;
      if (ok) ok = wait(&q_full[block.at], block.lap);
      unsigned long long mask[kBlocks][2];
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          mask[i][half] = ok ? masks[16 * i + row0 + 8 * half] : 0;
      // A node (at most kRows here) whose value holds infinities or NaN.
      const bool odd = __any_sync(0xffffffffu, ok && lane < sg.count && lane < kRows && flags[lane]);
      // Part `part` of a block's query rows, columns 16 ks ...
      auto load_q = [&](uint32_t (&a)[4], int i, int part, int ks) {
        ldsm4(a, ((q_at + q_lane) ^ (32 * (ks & 3))) + part * Sh::kQBytes + i * 16 * 128 +
                     (ks >> 2) * kRows * 128);
      };
      // The first part stays in registers where they hold it.
      constexpr bool kKeepQ = kBlocks == 1 || !kSplit;
      uint32_t qa[kBlocks][kKeepQ ? D / 16 : 1][4];
      if constexpr (kKeepQ) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) load_q(qa[i][ks], i, 0, ks);
      }

      float o[kBlocks][kCols / 8][4], m[kBlocks][2], l[kBlocks][2];
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        m[i][0] = m[i][1] = -INFINITY, l[i][0] = l[i][1] = 0.f;
#pragma unroll
        for (int c = 0; c < kCols / 8; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][c][j] = 0.f;
      }

      // This warp's 16 keys of a tile: scaled scores (base 2) of a block's rows row0,
      // row0 + 8 in s[0..3] (keys 2 quad, + 1) and s[4..7] (keys 8 + 2 quad, + 1),
      // -inf where unseen. Frees the keys; returns whether a reference has to
      // move.
      const int total = sg.length + sg.count;
      auto scores = [&](int tile, float (&s)[kBlocks][8]) {
        const int key0 = tile * kTile + 16 * warp;  // the warp's first
        const int ku = unit.at;
        if (ok) ok = wait(&full[ku], unit.lap);
        unit.next(units);
        float high[kBlocks][2][4], low[kBlocks][2][4];
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) high[i][h][j] = low[i][h][j] = 0.f;
        if (ok && key0 < total) {
          const uint32_t kt = ring + ku * Sh::kUnitBytes + k_lane;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t kb[4];
            ldsm4(kb, (kt ^ (32 * (ks & 3))) + (ks >> 2) * kTile * 128);
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) {
              if constexpr (!kKeepQ) load_q(qa[i][0], i, 0, ks);
              mma16816(high[i][0], qa[i][kKeepQ ? ks : 0], kb[0], kb[1]);
              mma16816(high[i][1], qa[i][kKeepQ ? ks : 0], kb[2], kb[3]);
              if constexpr (kSplit) {
                uint32_t a[4];
                load_q(a, i, 1, ks);
                mma16816(low[i][0], a, kb[0], kb[1]);
                mma16816(low[i][1], a, kb[2], kb[3]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[ku]);
        bool moves = false;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              s[i][4 * h + j] =
                  kSplit ? high[i][h][j] + low[i][h][j] : high[i][h][j] * p.scale_log2;
          if ((tile + 1) * kTile > sg.length) {
            // Behind the cached keys lie the nodes, behind them nothing.
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int age = key0 + 8 * (j >> 2) + 2 * quad + (j & 1) - sg.length;
              if (age >= 0 && (age >= sg.count || (mask[i][(j >> 1) & 1] >> age & 1) == 0))
                s[i][j] = -INFINITY;
            }
          }
          if constexpr (kWeights) {
            // Rows of scores end with a tile: what lies behind the last key is
            // written too, and not read.
            float* to = score_row(p, sg, row0) + key0 + 2 * quad;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (row0 + 8 * half < p.rows) {
                *reinterpret_cast<float2*>(to) = make_float2(s[i][2 * half], s[i][2 * half + 1]);
                *reinterpret_cast<float2*>(to + 8) =
                    make_float2(s[i][4 + 2 * half], s[i][5 + 2 * half]);
              }
              to += 8 * p.score_stride;
            }
          }
#pragma unroll
          for (int half = 0; half < 2; ++half)
            moves |= fmaxf(fmaxf(s[i][2 * half], s[i][2 * half + 1]),
                           fmaxf(s[i][4 + 2 * half], s[i][5 + 2 * half])) >
                     m[i][half] + kMoveThreshold;
        }
        return moves;
      };
      // The references move to the rows' largest scores so far.
      auto move = [&](const float (&s)[kBlocks][8]) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float top = fmaxf(fmaxf(s[i][2 * half], s[i][2 * half + 1]),
                              fmaxf(s[i][4 + 2 * half], s[i][5 + 2 * half]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (quad == 0) row_top[warp * kRows + 16 * i + row0 + 8 * half] = top;
          }
        sync_warps();
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float now = m[i][half];
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
              now = fmaxf(now, row_top[w * kRows + 16 * i + row0 + 8 * half]);
            const float a = now == m[i][half] ? 1.f : fast_exp2(m[i][half] - now);
            m[i][half] = now;
            l[i][half] *= a;
#pragma unroll
            for (int c = 0; c < kCols / 8; ++c) {
              o[i][c][2 * half] *= a;
              o[i][c][2 * half + 1] *= a;
            }
          }
      };
      // Probabilities are rounded to bf16 for the second product (2^-8 at most,
      // against an output in bf16 itself); their sum is not.
      auto publish = [&](const float (&s)[kBlocks][8]) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float ref = m[i][half] == -INFINITY ? 0.f : m[i][half];
            const float x0 = fast_exp2(s[i][2 * half] - ref);
            const float x1 = fast_exp2(s[i][2 * half + 1] - ref);
            const float x2 = fast_exp2(s[i][4 + 2 * half] - ref);
            const float x3 = fast_exp2(s[i][5 + 2 * half] - ref);
            l[i][half] += (x0 + x1) + (x2 + x3);
            uint8_t* row = smem + Sh::kOffP + parity * Sh::kPBytes + (2 * i + half) * 1024;
            *reinterpret_cast<uint32_t*>(row + p_store) = tc::bf16x2(x0, x1);
            *reinterpret_cast<uint32_t*>(row + (p_store ^ 16)) = tc::bf16x2(x2, x3);
          }
      };
      float s[kBlocks][8];
      if (total > 0) {
        const bool vote = scores(sg.tile0, s);
        if (sync_any(vote)) move(s);
        publish(s);
      }
      for (int tile = sg.tile0; tile < sg.tile1 && total > 0; ++tile) {
        const Turn values = unit;
        unit.next(units);
        const int key0 = tile * kTile, keys = min(kTile, total - key0);
        const bool edge = key0 + kTile > sg.length;
        if (keys < kTile) {
          // Behind the last node: zeros, for the product with zero
          // probabilities.
          if (ok) ok = wait(&full[values.at], values.lap);
          if (ok)
            for (int at = keys * (D / 8) + threadIdx.x; at < ((keys + 15) & ~15) * (D / 8);
                 at += 32 * kWarps)
              *reinterpret_cast<uint4*>(smem + Sh::kOffRing + values.at * Sh::kUnitBytes +
                                        tile_at(kTile, at / (D / 8), at % (D / 8))) =
                  make_uint4(0u, 0u, 0u, 0u);
          tc::fence_proxy_async();  // they come before the TMA's next writes
        }
        const bool more = tile + 1 < sg.tile1;
        const bool vote = more && scores(tile + 1, s);
        const bool moves = sync_any(vote);
        if (ok && keys == kTile) ok = wait(&full[values.at], values.lap);
        if (ok) {
          const uint32_t vt = ring + values.at * Sh::kUnitBytes;
          const uint32_t pt = base + Sh::kOffP + parity * Sh::kPBytes;
          auto weigh = [&](int ks) {  // 16 keys' probabilities and values
            uint32_t pa[kBlocks][4];
#pragma unroll
            for (int i = 0; i < kBlocks; ++i)
              ldsm4(pa[i], ((pt + q_lane) ^ (32 * ks)) + i * 16 * 128);
#pragma unroll
            for (int c = 0; c < kCols / 16; ++c) {
              uint32_t vb[4];
              ldsm4_t(vb, vt + v_lane[c] + ks * 16 * 128);
#pragma unroll
              for (int i = 0; i < kBlocks; ++i) {
                mma16816(o[i][2 * c], pa[i], vb[0], vb[1]);
                mma16816(o[i][2 * c + 1], pa[i], vb[2], vb[3]);
              }
            }
          };
          if (keys == kTile && !(edge && odd)) {
#pragma unroll
            for (int ks = 0; ks < kTile / 16; ++ks) weigh(ks);
          } else if (!(edge && odd)) {
            for (int ks = 0; 16 * ks < keys; ++ks) weigh(ks);
          } else {
            // A node's infinite or NaN value must not reach the nodes that do
            // not see it, as a product with zero would let it: key by key,
            // added only where it is visible.
#pragma unroll
            for (int j = 0; j < 2 * kBlocks; ++j) {
              const int i = j / 2, half = j % 2, r = 16 * i + row0 + 8 * half;
              for (int k = 0; k < keys; ++k) {
                const int age = key0 + k - sg.length;
                if (age >= 0 && (mask[i][half] >> age & 1) == 0) continue;
                const float w = __bfloat162float(*reinterpret_cast<const T*>(
                    smem + (pt - base) + r * 128 + (((k >> 3) ^ (r & 7)) << 4) + (k & 7) * 2));
#pragma unroll
                for (int c = 0; c < kCols / 8; ++c) {
                  const uint32_t v = *reinterpret_cast<const uint32_t*>(
                      smem + (vt - base) + tile_at(kTile, k, warp * (kCols / 8) + c) + 4 * quad);
                  o[i][c][2 * half] = fmaf(w, __uint_as_float(v << 16), o[i][c][2 * half]);
                  o[i][c][2 * half + 1] =
                      fmaf(w, __uint_as_float(v & 0xffff0000u), o[i][c][2 * half + 1]);
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[values.at]);
        parity ^= 1;
        if (more) {
          if (moves) move(s);
          publish(s);
        }
      }

      // The rows' sums, and the result: out, or to the workspace, whose parts
      // tree_finish.cu merges. (Two buffers: a segment without keys has
      // only this one barrier.)
      float* row_sum = row_sums + (n & 1) * kWarps * kRows;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float sum = l[i][half];
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if (quad == 0) row_sum[warp * kRows + 16 * i + row0 + 8 * half] = sum;
        }
      sync_warps();
      const bool whole = sg.whole();
      float* part = Parts<D>::mine(p, st);
#pragma unroll
      for (int j = 0; j < 2 * kBlocks; ++j) {
        const int i = j / 2, half = j % 2, r = 16 * i + row0 + 8 * half;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += row_sum[w * kRows + r];
        if (r >= p.rows) continue;
        if (whole) {
          const float f = 1.f / sum;
          if (kWeights && warp == 0 && quad == 0) write_lse(p, sg, r, m[i][half], sum);
          T* out = out_row<T>(p, sg.b, sg.h, r) + warp * kCols + 2 * quad;
#pragma unroll
          for (int c = 0; c < kCols / 8; ++c)
            *reinterpret_cast<uint32_t*>(out + 8 * c) =
                mask[i][half] == 0 ? 0u
                                   : tc::bf16x2(o[i][c][2 * half] * f, o[i][c][2 * half + 1] * f);
        } else {
          if (warp == 0 && quad == 0) part[r] = m[i][half], part[kRows + r] = sum;
#pragma unroll
          for (int c = 0; c < kCols / 8; ++c)
            *reinterpret_cast<float2*>(part +
                                       Parts<D>::at(p, r, warp * kCols + 8 * c + 2 * quad)) =
                make_float2(o[i][c][2 * half], o[i][c][2 * half + 1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[block.at]);
    }
  }
  if (!ok && lane == 0 && p.status) atomicOr(p.status, ASRBACK_STATUS_TIMEOUT);
}

template <int D, bool kSplit, int kBlocks, bool kWeights>
int launch(const TreeParams& p, cudaStream_t stream) {
  using Sh = Shape<D, kSplit, kBlocks>;
  auto kernel = tree_mma_kernel<D, kSplit, kBlocks, kWeights>;
  Maps maps;
  if (int rc = make_maps(&maps, p, D, kTile)) return rc;
  static thread_local int prepared_device = -1;
  int device = 0;
  if (int rc = check_cuda(cudaGetDevice(&device), "cudaGetDevice")) return rc;
  if (prepared_device != device) {
    if (int rc = check_cuda(
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kBudget),
            "cudaFuncSetAttribute(tree attention)"))
      return rc;
    prepared_device = device;
  }
  const int units = Sh::units(p.batch);
  return launch_pdl(kernel, dim3(p.ctas), dim3(kThreads), Sh::bytes(units, p.batch), stream,
                    "tree attention launch", maps, p, units);
}

template <int D, bool kSplit>
int launch(const TreeParams& p, cudaStream_t stream) {
  static_assert(kMaxWeightRows == 16, "weights come from one block");
  if constexpr (D == 64)
    if (p.block_rows == 32) return launch<D, kSplit, 2, false>(p, stream);
  return p.weights ? launch<D, kSplit, 1, true>(p, stream)
                   : launch<D, kSplit, 1, false>(p, stream);
}

}  // namespace

namespace tree {

int mma_ctas_per_sm(int head_dim, int block_rows) { return ctas_per_sm(head_dim, block_rows); }

int launch_mma(int head_dim, const TreeParams& p, cudaStream_t stream) {
  if (head_dim == 64) return p.q_norm ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
  return p.q_norm ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
}

}  // namespace tree
}  // namespace asrback
