// Draft-tree attention in bf16 for up to 64 query rows per block: mma.sync with a
// TMA warp, sm_100a. The split of the work is tree_attention.cu's.
//
// The call is bound by streaming the cache, so the TMA warp runs ahead of the
// products through the CTA's whole stretch, across items, and waits for nothing
// but a free ring unit (and once for the preparation kernel, which it overlaps
// with the first cached tiles). Roles:
//   the last   TMA: a segment's query block; a tile's keys, then its values,
//   warp       each one ring unit of 64 positions x D, in boxes of 32 positions
//              x 64 elements (128-byte swizzle), of a cut-off last tile only the
//              boxes that hold keys;
//   the others the products, four warps per group of 16 query rows. For the
//              scores each warp takes 16 of a tile's 64 keys; the probabilities
//              meet in shared memory, and for the output each warp takes a
//              quarter of the columns, over all keys: no merge of outputs
//              between warps, and a quarter of its registers.
// One barrier per tile among a group's warps: the scores of tile t + 1 are
// computed before it, so that the barrier which publishes tile t's
// probabilities also votes on whether a row of tile t + 1 passes its softmax
// reference by more than 8 (base 2); only then the references move.
//
// mma.sync instead of tcgen05: it issues 1000 multiply-adds per cycle and SM
// (measured: one m16n8k16 in 2.05 cycles), enough for 64 rows of head_dim 128 at
// the rate the cache arrives, while a 128-row tcgen05 tile would be mostly empty
// and its softmax would run in a few lanes of one warp.
#include <type_traits>

#include "tcgen05.cuh"
#include "tree_attention.cuh"

namespace asrback {
namespace {

using namespace tree;

constexpr int kGroupWarps = 4;
constexpr int kGroupThreads = 32 * kGroupWarps;
constexpr int kBoxKeys = 32;
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
// Barrier among a group's warps that tells all whether any thread voted.
__device__ __forceinline__ bool group_any(int id, bool vote) {
  uint32_t any;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %1, 0;\n"
      "barrier.cta.red.or.pred q, %2, 128, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(any)
      : "r"(vote ? 1u : 0u), "r"(id)
      : "memory");
  return any != 0;
}

// CTAs per SM: as many as registers and shared memory allow, since a tile's
// chain of products, barrier and exponentials and an item's end are latencies
// that only other CTAs' work fills.
constexpr int ctas_per_sm(int head_dim, int groups) {
  return groups == 1 ? (head_dim == 64 ? 4 : 3) : groups == 2 ? 2 : 1;
}

template <int D, int G, bool kSplit>  // G: groups of 16 query rows
struct Shape {
  static constexpr int kRows = 16 * G;
  static constexpr int kThreads = kGroupThreads * G + 32;
  static constexpr int kPerSm = ctas_per_sm(D, G);
  static constexpr int kUnitBytes = kTile * D * 2;  // keys or values of a tile
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kBlockBytes = (kSplit ? 2 : 1) * kQBytes + kRows * 8;
  static constexpr int kSlotBytes = (kBlockBytes + 127) / 128 * 128;
  // With many CTAs per SM ring units are worth more than a second block.
  static constexpr int kQSlots = kPerSm > 2 ? 1 : 2;
  static constexpr int kOffP = kQSlots * kSlotBytes;  // [2][rows][64 keys]
  static constexpr int kPBytes = kRows * kTile * 2;
  static constexpr int kOffRing = (kOffP + 2 * kPBytes + 1023) / 1024 * 1024;
  // row_top, row_sum[2], scratch, flags, barriers, then the tile list; slack to
  // align the base to 1024.
  static constexpr int kMisc = 3 * kGroupWarps * kRows * 4 + 128 + 64 + (2 * kMaxUnits + 4) * 8;
  static constexpr int kBudget = (228 * 1024 / kPerSm - 1024) / 16 * 16;
  static constexpr int units(int batch) {
    const int n = (kBudget - 1024 - kOffRing - kMisc - list_bytes(batch)) / kUnitBytes;
    return n > kMaxUnits ? kMaxUnits : n;
  }
  static constexpr int bytes(int units, int batch) {
    return 1024 + kOffRing + units * kUnitBytes + kMisc + list_bytes(batch);
  }
  // A tile's keys are read before the last tile's values: three units make
  // progress, a fourth keeps a load in flight.
  static_assert(units(kMaxBatch) >= 3, "the ring is too short");
};

template <int D, int G, bool kSplit, bool kWeights>
__global__ void __launch_bounds__(Shape<D, G, kSplit>::kThreads, Shape<D, G, kSplit>::kPerSm)
    tree_mma_kernel(const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TreeParams p,
                    const int units) {
  using Sh = Shape<D, G, kSplit>;
  using T = __nv_bfloat16;
  constexpr int kRows = Sh::kRows, kThreads = Sh::kThreads, kQSlots = Sh::kQSlots;
  constexpr int kCols = D / kGroupWarps;  // output columns of a warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* misc = smem + Sh::kOffRing + units * Sh::kUnitBytes;
  float* row_top = reinterpret_cast<float*>(misc);                   // [warp of group][rows]
  float* row_sums = row_top + kGroupWarps * kRows;                   // [2][warp of group][rows]
  int* scratch = reinterpret_cast<int*>(row_sums + 2 * kGroupWarps * kRows);  // [32]
  int* is_last = scratch + 32;                                       // [group]
  int* odd_values = is_last + 8;                                     // [group]
  uint64_t* full = reinterpret_cast<uint64_t*>(is_last + 16);        // [unit]
  uint64_t* empty = full + kMaxUnits;
  uint64_t* q_full = empty + kMaxUnits;  // [slot]
  uint64_t* q_empty = q_full + kQSlots;
  TileList list(misc + Sh::kMisc, p.batch);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int u = 0; u < units; ++u) {
      mbar_init(&full[u], 1);
      mbar_init(&empty[u], kGroupWarps * G);
    }
    for (int s = 0; s < kQSlots; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], kGroupWarps * G);
    }
    fence_barrier_init();
  }
  if (threadIdx.x < G) odd_values[threadIdx.x] = -1;
  griddep_launch_dependents();
  // The lengths and counts are older than the preparation kernel, which began
  // behind them: only what that kernel writes is waited for, further down.
  Stretch st = begin_stretch<kThreads>(p, list, scratch);  // has a barrier: inits are visible
  const Segment& sg = st.seg;
  auto wait = [](uint64_t* bar, int parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity & 1)) != 0;
  };
  bool ok = true;

  if (warp == kGroupWarps * G) {
    // ------------------------------------------------------------------- TMA
    const bool leader = tc::elect_one();
    if (leader) {
      tc::prefetch_tensormap(&map_k);
      tc::prefetch_tensormap(&map_v);
    }
    __syncwarp();
    const uint64_t policy = l2_evict_first_policy();
    bool waited = false;
    int unit = 0, lap = 0;
    for (int n = 0; ok && next_segment(p, list, st); ++n) {
      // The query block is loaded as soon as its buffer is free, and at the
      // latest when the products could not go on without it: before the ring
      // waits for a unit that this segment itself has filled.
      const int slot = n % kQSlots, q_lap = n / kQSlots;
      bool q_due = true;
      auto load_q = [&](bool now) {
        if (!q_due || (!now && !waited)) return;
        if (!waited) griddep_wait();
        waited = true;
        if (q_lap > 0) {
          if (!now && !__all_sync(0xffffffffu, mbar_test(&q_empty[slot], (q_lap - 1) & 1))) return;
          ok = wait(&q_empty[slot], q_lap - 1);
        }
        q_due = false;
        if (ok && leader) {
          mbar_arrive_expect_tx(&q_full[slot], Sh::kBlockBytes);
          bulk_g2s(smem + slot * Sh::kSlotBytes, p.q_blocks + (int64_t)sg.item * Sh::kBlockBytes,
                   Sh::kBlockBytes, &q_full[slot], policy);
        }
        __syncwarp();
      };
      const int total = sg.length + sg.count;
      int filled = 0;  // units of this segment
      for (int tile = sg.tile0; tile < sg.tile1 && ok && total > 0; ++tile) {
        const int boxes = (min(kTile, total - tile * kTile) + kBoxKeys - 1) / kBoxKeys;
        // A tile with nodes in it comes after the preparation.
        if (!waited && tile * kTile + boxes * kBoxKeys > sg.length) load_q(true);
        for (int which = 0; which < 2 && ok; ++which, ++filled) {
          load_q(filled >= units);
          if (ok && lap > 0) ok = wait(&empty[unit], lap - 1);
          if (ok && leader) {
            uint8_t* dst = smem + Sh::kOffRing + unit * Sh::kUnitBytes;
            mbar_arrive_expect_tx(&full[unit], boxes * kBoxKeys * D * 2);
            for (int box = 0; box < boxes; ++box)
#pragma unroll
              for (int c = 0; c < D / 64; ++c)
                tc::tma_load_4d(dst + c * kTile * 128 + box * kBoxKeys * 128,
                                which ? &map_v : &map_k, 64 * c, tile * kTile + box * kBoxKeys,
                                sg.h, sg.b, &full[unit]);
          }
          __syncwarp();
          if (ok && ++unit == units) unit = 0, ++lap;
        }
      }
      if (ok) load_q(true);
    }
    // A wait gave up: the copies in flight still have to land before the CTA
    // may end.
    if (!ok)
      for (int u = 0; u < units; ++u) {
        const int laps = lap + (u < unit ? 1 : 0);
        if (laps > 0) wait(&full[u], laps - 1);
      }
  } else {
    // -------------------------------------------------------------- products
    const int group = warp / kGroupWarps, gw = warp % kGroupWarps;
    const int gtid = threadIdx.x - group * kGroupThreads;
    const int barrier = 1 + group;
    const int quad = lane & 3, row0 = 16 * group + (lane >> 2);  // rows row0 and row0 + 8
    const int mat = lane >> 3, mrow = lane & 7;  // ldmatrix: lane l gives row l % 8 of matrix l / 8
    const uint32_t base = smem_addr(smem);
    int unit = 0, lap = 0, n = 0;
    auto advance = [&] {
      if (++unit == units) unit = 0, ++lap;
    };
    for (; next_segment(p, list, st); ++n) {
      const int slot = n % kQSlots;
      const uint32_t q_at = base + slot * Sh::kSlotBytes;
      const auto* masks = reinterpret_cast<const unsigned long long*>(
          smem + slot * Sh::kSlotBytes + Sh::kBlockBytes - kRows * 8);
      if (ok) ok = wait(&q_full[slot], n / kQSlots);
      const unsigned long long mask[2] = {ok ? masks[row0] : 0, ok ? masks[row0 + 8] : 0};
      uint32_t qa[D / 16][4];
      auto load_q = [&](uint32_t (&a)[4], int part, int ks) {
        ldsm4(a, q_at + part * Sh::kQBytes +
                     tile_at<D>(kRows, 16 * group + (mat & 1) * 8 + mrow, 2 * ks + (mat >> 1)));
      };
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) load_q(qa[ks], 0, ks);

      float o[kCols / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kCols / 8; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[c][j] = 0.f;

      // This warp's 16 keys of a tile: scaled scores (base 2) of rows row0,
      // row0 + 8 in s[0..3] (keys 2 quad, + 1) and s[4..7] (keys 8 + 2 quad, + 1),
      // -inf where unseen. Frees the keys; returns whether a reference has to
      // move.
      const int total = sg.length + sg.count;
      auto scores = [&](int tile, float (&s)[8]) {
        const int key0 = tile * kTile + 16 * gw;  // the warp's first
        const int ku = unit, klap = lap;
        advance();
        if (ok) ok = wait(&full[ku], klap);
        float high[2][4], low[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) high[h][j] = low[h][j] = 0.f;
        if (ok && key0 < total) {
          const uint32_t kt = base + Sh::kOffRing + ku * Sh::kUnitBytes;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t kb[4];
            ldsm4(kb, kt + tile_at<D>(kTile, 16 * gw + (mat >> 1) * 8 + mrow, 2 * ks + (mat & 1)));
            mma16816(high[0], qa[ks], kb[0], kb[1]);
            mma16816(high[1], qa[ks], kb[2], kb[3]);
            if constexpr (kSplit) {
              uint32_t a[4];
              load_q(a, 1, ks);
              mma16816(low[0], a, kb[0], kb[1]);
              mma16816(low[1], a, kb[2], kb[3]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[ku]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s[4 * h + j] = kSplit ? high[h][j] + low[h][j] : high[h][j] * p.scale_log2;
        if ((tile + 1) * kTile > sg.length) {
          // Behind the cached keys lie the nodes, behind them nothing.
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = key0 + 8 * (i >> 2) + 2 * quad + (i & 1);
            const int age = key - sg.length;
            if (age >= 0 && (age >= sg.count || (mask[(i >> 1) & 1] >> age & 1) == 0))
              s[i] = -INFINITY;
          }
        }
        if constexpr (kWeights) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = row0 + 8 * ((i >> 1) & 1), key = key0 + 8 * (i >> 2) + 2 * quad + (i & 1);
            if (r < p.rows && key < total) score_row(p, sg, r)[key] = s[i];
          }
        }
        const float limit0 = m[0] + kMoveThreshold, limit1 = m[1] + kMoveThreshold;
        return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[4], s[5])) > limit0 ||
               fmaxf(fmaxf(s[2], s[3]), fmaxf(s[6], s[7])) > limit1;
      };
      // The references move to the rows' largest scores so far.
      auto move = [&](const float (&s)[8]) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float top = fmaxf(fmaxf(s[2 * half], s[2 * half + 1]),
                            fmaxf(s[4 + 2 * half], s[5 + 2 * half]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          if (quad == 0) row_top[gw * kRows + row0 + 8 * half] = top;
        }
        named_sync(barrier, kGroupThreads);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float now = m[half];
#pragma unroll
          for (int w = 0; w < kGroupWarps; ++w)
            now = fmaxf(now, row_top[w * kRows + row0 + 8 * half]);
          const float a = now == m[half] ? 1.f : fast_exp2(m[half] - now);
          m[half] = now;
          l[half] *= a;
#pragma unroll
          for (int c = 0; c < kCols / 8; ++c) {
            o[c][2 * half] *= a;
            o[c][2 * half + 1] *= a;
          }
        }
      };
      // Probabilities are rounded to bf16 for the second product (2^-8 at most,
      // against an output in bf16 itself); their sum is not.
      auto publish = [&](int parity, const float (&s)[8]) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = row0 + 8 * half;
          const float ref = m[half] == -INFINITY ? 0.f : m[half];
          const float x0 = fast_exp2(s[2 * half] - ref), x1 = fast_exp2(s[2 * half + 1] - ref);
          const float x2 = fast_exp2(s[4 + 2 * half] - ref), x3 = fast_exp2(s[5 + 2 * half] - ref);
          l[half] += (x0 + x1) + (x2 + x3);
          uint8_t* row = smem + Sh::kOffP + parity * Sh::kPBytes + r * 128 + 4 * quad;
          *reinterpret_cast<uint32_t*>(row + (((2 * gw) ^ (r & 7)) << 4)) = tc::bf16x2(x0, x1);
          *reinterpret_cast<uint32_t*>(row + (((2 * gw + 1) ^ (r & 7)) << 4)) = tc::bf16x2(x2, x3);
        }
      };
      // Values of a tile that reaches behind the cached keys, this warp's 16
      // keys: zeros behind the last node, for the product with zero
      // probabilities; notes a node's infinite or NaN value.
      auto inspect = [&](int tile, int vu, int vlap) {
        if (ok) ok = wait(&full[vu], vlap);
        if (!ok) return;
        bool odd = false;
        for (int i = lane; i < 16 * (D / 8); i += 32) {
          const int row = 16 * gw + i / (D / 8), age = tile * kTile + row - sg.length;
          if (age < 0) continue;
          uint4* at = reinterpret_cast<uint4*>(smem + Sh::kOffRing + vu * Sh::kUnitBytes +
                                               tile_at<D>(kTile, row, i % (D / 8)));
          if (age >= sg.count) {
            if (group == 0) *at = make_uint4(0u, 0u, 0u, 0u);
          } else {
            const uint4 v = *at;
            const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              odd |= (words[j] & 0x7f80u) == 0x7f80u || (words[j] & 0x7f800000u) == 0x7f800000u;
          }
        }
        if (__any_sync(0xffffffffu, odd) && lane == 0) odd_values[group] = n;
        tc::fence_proxy_async();  // the zeros come before the TMA's next writes
      };

      float s[8];
      if (total > 0) {
        const bool vote = scores(sg.tile0, s);
        if (group_any(barrier, vote)) move(s);
        publish(0, s);
      }
      for (int tile = sg.tile0; tile < sg.tile1 && total > 0; ++tile) {
        const int parity = (tile - sg.tile0) & 1;
        const int vu = unit, vlap = lap;
        advance();
        const bool edge = (tile + 1) * kTile > sg.length;
        if (edge) {
          inspect(tile, vu, vlap);
          // The zeros are the first group's; every group reads them.
          if (G > 1) named_sync(8, kGroupThreads * G);
        }
        const bool more = tile + 1 < sg.tile1;
        const bool vote = more && scores(tile + 1, s);
        const bool moves = group_any(barrier, vote);
        if (ok && !edge) ok = wait(&full[vu], vlap);
        if (ok) {
          const uint32_t vt = base + Sh::kOffRing + vu * Sh::kUnitBytes;
          const uint32_t pt = base + Sh::kOffP + parity * Sh::kPBytes;
          if (!edge || odd_values[group] != n) {
            const int steps = min(kTile, (total - tile * kTile + 15) & ~15) / 16;
#pragma unroll
            for (int ks = 0; ks < kTile / 16; ++ks) {
              if (ks >= steps) break;
              uint32_t pa[4];
              const int r = 16 * group + (mat & 1) * 8 + mrow;
              ldsm4(pa, pt + r * 128 + (((2 * ks + (mat >> 1)) ^ (r & 7)) << 4));
#pragma unroll
              for (int c = 0; c < kCols / 16; ++c) {
                uint32_t vb[4];
                ldsm4_t(vb, vt + tile_at<D>(kTile, 16 * ks + (mat & 1) * 8 + mrow,
                                            gw * (kCols / 8) + 2 * c + (mat >> 1)));
                mma16816(o[2 * c], pa, vb[0], vb[1]);
                mma16816(o[2 * c + 1], pa, vb[2], vb[3]);
              }
            }
          } else {
            // A node's infinite or NaN value must not reach the nodes that do
            // not see it, as a product with zero would let it: key by key,
            // added only where it is visible.
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int r = row0 + 8 * half;
              for (int k = 0; k < min(kTile, total - tile * kTile); ++k) {
                const int age = tile * kTile + k - sg.length;
                if (age >= 0 && (mask[half] >> age & 1) == 0) continue;
                const float w = __bfloat162float(*reinterpret_cast<const T*>(
                    smem + (pt - base) + r * 128 + (((k >> 3) ^ (r & 7)) << 4) + (k & 7) * 2));
#pragma unroll
                for (int c = 0; c < kCols / 8; ++c) {
                  const uint32_t v = *reinterpret_cast<const uint32_t*>(
                      smem + (vt - base) + tile_at<D>(kTile, k, gw * (kCols / 8) + c) + 4 * quad);
                  o[c][2 * half] = fmaf(w, __uint_as_float(v << 16), o[c][2 * half]);
                  o[c][2 * half + 1] =
                      fmaf(w, __uint_as_float(v & 0xffff0000u), o[c][2 * half + 1]);
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[vu]);
        if (more) {
          if (moves) move(s);
          publish(parity ^ 1, s);
        }
      }

      // The rows' sums, and the result: out, or to the workspace for the
      // item's last CTA to merge. (Two buffers: a segment without keys has
      // only this one barrier.)
      float* row_sum = row_sums + (n & 1) * kGroupWarps * kRows;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float sum = l[half];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (quad == 0) row_sum[gw * kRows + row0 + 8 * half] = sum;
      }
      named_sync(barrier, kGroupThreads);
      const bool whole = sg.first_cta == sg.last_cta;
      float* part = Parts<D, kRows>::mine(p, st);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = row0 + 8 * half, row = sg.mblock * kRows + r;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kGroupWarps; ++w) sum += row_sum[w * kRows + r];
        if (row >= p.rows) continue;
        if (whole) {
          const float f = 1.f / sum;
          if (p.weights && gw == 0 && quad == 0)
            p.lse[((int64_t)sg.b * p.kv_heads + sg.h) * p.rows + row] =
                mask[half] == 0 ? INFINITY : m[half] + log2f(sum);
          T* out = static_cast<T*>(p.out) + sg.b * p.o_sb + (row / p.group) * p.o_sn +
                   (sg.h * p.group + row % p.group) * p.o_sh + gw * kCols + 2 * quad;
#pragma unroll
          for (int c = 0; c < kCols / 8; ++c)
            *reinterpret_cast<uint32_t*>(out + 8 * c) =
                mask[half] == 0 ? 0u : tc::bf16x2(o[c][2 * half] * f, o[c][2 * half + 1] * f);
        } else {
          if (gw == 0 && quad == 0) part[r] = m[half], part[kRows + r] = sum;
#pragma unroll
          for (int c = 0; c < kCols / 8; ++c)
            *reinterpret_cast<float2*>(part + 2 * kRows + r * D + gw * kCols + 8 * c + 2 * quad) =
                make_float2(o[c][2 * half], o[c][2 * half + 1]);
        }
      }
      if (!whole) {
        __threadfence();
        named_sync(barrier, kGroupThreads);
        if (gtid == 0) is_last[group] = take_ticket(sg, p.counters + sg.item * G + group);
        named_sync(barrier, kGroupThreads);
        if (is_last[group] && ok) {
          __threadfence();
          merge_parts<D, kRows, 16, kGroupThreads, T>(p, st, masks, 16 * group, gtid);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[slot]);
    }
  }
  if (!ok && lane == 0 && p.status) atomicOr(p.status, ASRBACK_STATUS_TIMEOUT);
}

// The cache as a 4-D map {d, position, head, row}, box 64 x kBoxKeys x 1 x 1.
int make_map(CUtensorMap* map, void* base, const TreeParams& p, int head_dim) {
  int rc = ASRBACK_OK;
  auto encode = tc::tensor_map_encoder(&rc);
  if (!encode) return rc;
  // A dimension of one may have any stride; the encoder wants a plausible one.
  const auto bytes = [&](int64_t stride, int64_t size) {
    return static_cast<cuuint64_t>((size > 1 ? stride : head_dim) * 2);
  };
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)p.cache_length,
                              (cuuint64_t)p.kv_heads, (cuuint64_t)p.batch};
  const cuuint64_t strides[3] = {bytes(p.c_sp, p.cache_length), bytes(p.c_sh, p.kv_heads),
                                 bytes(p.c_sb, p.batch)};
  const cuuint32_t box[4] = {64, kBoxKeys, 1, 1}, ones[4] = {1, 1, 1, 1};
  const CUresult res =
      encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides, box, ones,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (res != CUDA_SUCCESS)
    return fail(ASRBACK_ERR_ARGUMENT,
                "cuTensorMapEncodeTiled rejected the cache (error %d): strides (%lld, %lld, %lld)",
                (int)res, (long long)p.c_sb, (long long)p.c_sp, (long long)p.c_sh);
  return ASRBACK_OK;
}

template <int D, int G, bool kSplit, bool kWeights>
int launch(const TreeParams& p, cudaStream_t stream) {
  using Sh = Shape<D, G, kSplit>;
  auto kernel = tree_mma_kernel<D, G, kSplit, kWeights>;
  CUtensorMap map_k, map_v;
  if (int rc = make_map(&map_k, p.key_cache, p, D)) return rc;
  if (int rc = make_map(&map_v, p.value_cache, p, D)) return rc;
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
  return launch_pdl(kernel, dim3(p.ctas), dim3(Sh::kThreads), Sh::bytes(units, p.batch), stream,
                    "tree attention launch", map_k, map_v, p, units);
}

template <int D, bool kSplit>
int pick(int block_rows, const TreeParams& p, cudaStream_t stream) {
  if (p.weights) return launch<D, 1, kSplit, true>(p, stream);
  if (block_rows == 16) return launch<D, 1, kSplit, false>(p, stream);
  if (block_rows == 32) return launch<D, 2, kSplit, false>(p, stream);
  return launch<D, 4, kSplit, false>(p, stream);
}

}  // namespace

namespace tree {

int mma_ctas_per_sm(int head_dim, int block_rows) { return ctas_per_sm(head_dim, block_rows / 16); }

int launch_mma(int head_dim, int block_rows, const TreeParams& p, cudaStream_t stream) {
  if (head_dim == 64)
    return p.q_norm ? pick<64, true>(block_rows, p, stream) : pick<64, false>(block_rows, p, stream);
  return p.q_norm ? pick<128, true>(block_rows, p, stream) : pick<128, false>(block_rows, p, stream);
}

}  // namespace tree
}  // namespace asrback
