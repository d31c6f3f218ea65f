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
// the rows' lengths, so all CTAs stream the same number of bytes. A stretch
// that covers only part of an item leaves its unnormalised result (m, l, o) in
// the workspace; the last CTA of the item to finish (an atomic ticket that it
// re-arms) merges the parts in list order, so results do not depend on which
// CTA was last.
//
// The tree is an item's last tile. Its keys and values come from the call's
// inputs, not from the cache: the CTA that owns the tile normalises and
// rotates them, writes them to the cache and uses them from shared memory, so
// no CTA waits for another's cache write.
#include "../../include/asrback_attn.h"
#include "capi_internal.h"
#include "common.cuh"
#include "tree_attention.cuh"

#include <algorithm>
#include <type_traits>

namespace asrback {
namespace {

using namespace tree;

// ----------------------------------------------------------- bf16, mma.sync
//
// Four warps; a warp owns 16 of a tile's 64 keys and all the block's query
// rows (16 or 32), with its own softmax state, its own part of the ring and
// no barrier with the other warps until the end of a stretch.

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
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes global to shared, or 16 zero bytes where `valid` is false.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// Byte offset of 16-byte piece `piece` of row `row` in a [rows][D] bf16 tile:
// pieces permuted within a row so that eight rows' same piece (an ldmatrix
// phase) and one row's pieces (a copy) both touch all banks once.
template <int D>
__device__ __forceinline__ int swz(int row, int piece) {
  return row * (D * 2) + ((piece ^ (row & 7)) << 4);
}

template <int D, int MT, bool kWeights>
struct MmaShape {
  static constexpr int kRows = 16 * MT;
  static constexpr int kStages = 3;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kRingBytes = kStages * 2 * kTileBytes;  // [stage][keys, values], at 0
  static constexpr int kOffQ = kRingBytes;  // q rounded to bf16; then, with weights, the rest
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kOffCommon = kOffQ + (kWeights ? 2 : 1) * kQBytes;
  static constexpr int kSmem = kOffCommon + (int)sizeof(Common<kRows>);
  // The warps' results at the end of a stretch, in the ring.
  static constexpr int kMergeFloats = 4 * kRows * (D + 2);
  static_assert(kMergeFloats * 4 <= kRingBytes, "the merge buffer must fit the ring");
};

template <int D, int MT, bool kWeights>
__global__ void __launch_bounds__(kThreads, MT == 1 ? 2 : 1)
    tree_mma_kernel(const __grid_constant__ TreeParams p) {
  using Sh = MmaShape<D, MT, kWeights>;
  using T = __nv_bfloat16;
  constexpr int kRows = Sh::kRows, kStages = Sh::kStages;
  constexpr int kPieces = D / 8;             // 16-byte pieces of a row
  constexpr int kPasses = 16 * kPieces / 32;  // copies per lane for 16 rows
  constexpr int kRowStep = 32 / kPieces;      // rows between a lane's copies
  extern __shared__ __align__(1024) uint8_t smem[];
  auto& cm = *reinterpret_cast<Common<kRows>*>(smem + Sh::kOffCommon);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane & 3, group_row = lane >> 2;

  griddep_wait();
  griddep_launch_dependents();
  Stretch st = begin_stretch(p, cm);
  const uint32_t ring = smem_addr(smem);
  const uint32_t q_smem = smem_addr(smem + Sh::kOffQ);
  // ldmatrix addresses: lane l gives row l % 8 of matrix l / 8.
  const int mat = lane >> 3, mrow = lane & 7;

  while (next_segment(p, cm, st)) {
    const Segment& sg = st.seg;
    // Query rows of the block: normalised, rotated, rounded once to bf16. With
    // weights, q = hi + lo in two bf16 parts, since a rounding of q to 8 bits
    // would put 2^-9 * |s| into every accumulated weight.
    prepare_rows<D, kRows, T>(p, sg, cm, warp, lane, [&](int r, int e, const float* x, int n) {
      uint8_t* hi = smem + Sh::kOffQ + swz<D>(r, e / 8) + (e % 8) * 2;
#pragma unroll
      for (int j = 0; j < n; j += 2) {
        const uint32_t h = bf16_pair(x[j], x[j + 1]);
        *reinterpret_cast<uint32_t*>(hi + 2 * j) = h;
        if constexpr (kWeights)
          *reinterpret_cast<uint32_t*>(hi + Sh::kQBytes + 2 * j) =
              bf16_pair(x[j] - __uint_as_float(h << 16), x[j + 1] - __uint_as_float(h & 0xffff0000u));
      }
    });
    __syncthreads();
    uint32_t qa[MT][D / 16][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
        ldsm4(qa[t][ks], q_smem + swz<D>(16 * t + (mat & 1) * 8 + mrow, 2 * ks + (mat >> 1)));

    float o[MT][D / 8][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[t][n][j] = 0.f;
    }

    const T* kbase = static_cast<const T*>(p.key_cache) + sg.b * p.c_sb + sg.h * p.c_sh;
    const T* vbase = static_cast<const T*>(p.value_cache) + sg.b * p.c_sb + sg.h * p.c_sh;
    const int copy_row = lane / kPieces, copy_piece = lane % kPieces;
    auto copy_tile = [&](int stage, int tile) {
      const uint32_t dst = ring + stage * 2 * Sh::kTileBytes;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int row = 16 * warp + copy_row + i * kRowStep;
        const int key = tile * kTile + row;
        const bool in = key < sg.length;
        const int64_t at = (int64_t)(in ? key : 0) * p.c_sp + copy_piece * 8;
        cp_async16(dst + swz<D>(row, copy_piece), kbase + at, in);
        cp_async16(dst + Sh::kTileBytes + swz<D>(row, copy_piece), vbase + at, in);
      }
    };

    // One warp's 16 keys against the block's rows. `visible(t, row half, key in
    // the tile)` masks; kMask is off for full cache tiles.
    // `finite` is false only where a node's value is not.
    auto compute = [&](int stage, auto masked, int first_key, bool finite, auto visible) {
      constexpr bool kMask = decltype(masked)::value;
      const uint32_t kt = ring + stage * 2 * Sh::kTileBytes, vt = kt + Sh::kTileBytes;
      float s[MT][2][4];
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[t][n][j] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t kb[4];
        ldsm4(kb, kt + swz<D>(16 * warp + (mat >> 1) * 8 + mrow, 2 * ks + (mat & 1)));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          mma16816(s[t][0], qa[t][ks], kb[0], kb[1]);
          mma16816(s[t][1], qa[t][ks], kb[2], kb[3]);
          if constexpr (kWeights) {
            uint32_t lo[4];
            ldsm4(lo, q_smem + Sh::kQBytes +
                          swz<D>(16 * t + (mat & 1) * 8 + mrow, 2 * ks + (mat >> 1)));
            mma16816(s[t][0], lo, kb[0], kb[1]);
            mma16816(s[t][1], lo, kb[2], kb[3]);
          }
        }
      }
      uint32_t pa[MT][4];
      bool moved = false;
      float alpha[MT][2];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float top = -INFINITY;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float& x = s[t][n][2 * half + j];
              x *= p.scale_log2;
              if constexpr (kMask) {
                if (!visible(16 * t + 8 * half + group_row, 16 * warp + 8 * n + 2 * quad + j))
                  x = -INFINITY;
              }
              top = fmaxf(top, x);
            }
          if constexpr (kWeights) {
            const int r = 16 * t + 8 * half + group_row;
            if (r < p.rows) {
              float* out = score_row(p, sg, r) + first_key + 16 * warp + 2 * quad;
#pragma unroll
              for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                  if (!kMask || 16 * warp + 8 * n + 2 * quad + j < sg.tile_keys(first_key))
                    out[8 * n + j] = s[t][n][2 * half + j];
            }
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float now = fmaxf(m[t][half], top);
          const float ref = now == -INFINITY ? 0.f : now;
          alpha[t][half] = fast_exp2(m[t][half] - ref);
          moved |= now != m[t][half];
          m[t][half] = now;
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float& x = s[t][n][2 * half + j];
              x = fast_exp2(x - ref);
              sum += x;
            }
          l[t][half] = l[t][half] * alpha[t][half] + sum;
        }
        // Probabilities are rounded to bf16 for the second product: 2^-9 apart
        // at most, against an output rounded to bf16 itself; their sum is not.
        pa[t][0] = bf16_pair(s[t][0][0], s[t][0][1]);
        pa[t][1] = bf16_pair(s[t][0][2], s[t][0][3]);
        pa[t][2] = bf16_pair(s[t][1][0], s[t][1][1]);
        pa[t][3] = bf16_pair(s[t][1][2], s[t][1][3]);
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[t][n][j] *= alpha[t][j >> 1];
      }
      if (!kMask || finite) {
#pragma unroll
        for (int dp = 0; dp < D / 16; ++dp) {
          uint32_t vb[4];
          ldsm4_t(vb, vt + swz<D>(16 * warp + (mat & 1) * 8 + mrow, 2 * dp + (mat >> 1)));
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            mma16816(o[t][2 * dp], pa[t], vb[0], vb[1]);
            mma16816(o[t][2 * dp + 1], pa[t], vb[2], vb[3]);
          }
        }
      }
      if constexpr (kMask) {
        if (finite) return;
        // A node's infinite or NaN value must not reach the nodes that do not
        // see it, as a product with zero would let it: one key at a time,
        // added only where it is visible.
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            for (int key = 0; key < 16; ++key) {
              // Key `key` of the warp lies in half key % 2 of a register of
              // the quad's lane (key % 8) / 2.
              const uint32_t pair = __shfl_sync(
                  0xffffffffu, key < 8 ? pa[t][half] : pa[t][2 + half], (lane & ~3) | ((key & 7) >> 1));
              const float w = __uint_as_float(key & 1 ? pair & 0xffff0000u : pair << 16);
              if (!visible(16 * t + 8 * half + group_row, 16 * warp + key)) continue;
#pragma unroll
              for (int n = 0; n < D / 8; ++n) {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(
                    smem + (vt - ring) + swz<D>(16 * warp + key, n) + 4 * quad);
                o[t][n][2 * half] = fmaf(w, __uint_as_float(v << 16), o[t][n][2 * half]);
                o[t][n][2 * half + 1] =
                    fmaf(w, __uint_as_float(v & 0xffff0000u), o[t][n][2 * half + 1]);
              }
            }
      }
    };

    // The stretch's cache tiles, kStages - 1 in flight.
    const int last = min(sg.tile1, sg.tiles - 1);  // one past the last cache tile
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
      if (sg.tile0 + s < last) copy_tile(s, sg.tile0 + s);
      cp_commit();
    }
    int stage = 0;
    for (int tile = sg.tile0; tile < last; ++tile) {
      cp_wait<kStages - 2>();
      __syncwarp();
      const int ahead = tile + kStages - 1;
      if (ahead < last) copy_tile(stage == 0 ? kStages - 1 : stage - 1, ahead);
      cp_commit();
      if ((tile + 1) * kTile <= sg.length)
        compute(stage, std::false_type{}, tile * kTile, true, [](int, int) { return true; });
      else
        compute(stage, std::true_type{}, tile * kTile, true,
                [&](int, int key) { return tile * kTile + key < sg.length; });
      __syncwarp();
      stage = stage == kStages - 1 ? 0 : stage + 1;
    }

    // The tree's own tile.
    if (sg.tile1 == sg.tiles && sg.count > 0) {
      __syncthreads();  // every warp is done with its part of stage 0
      const bool finite = load_tree_tile<D, T>(
          p, sg, cm, warp, lane, [&](int i, int e, const float* k, const float* v, int n) {
            uint8_t* dst = smem + swz<D>(i, e / 8) + (e % 8) * 2;
#pragma unroll
            for (int j = 0; j < n; j += 2) {
              *reinterpret_cast<uint32_t*>(dst + 2 * j) = bf16_pair(k[j], k[j + 1]);
              *reinterpret_cast<uint32_t*>(dst + Sh::kTileBytes + 2 * j) =
                  bf16_pair(v[j], v[j + 1]);
            }
          });
      if (16 * warp < sg.count)
        compute(0, std::true_type{}, sg.length, finite,
                [&](int r, int key) { return (cm.mask[r] >> key & 1) != 0; });
    }

    // The four warps' states become one.
    __syncthreads();
    float* part_m = reinterpret_cast<float*>(smem);  // [warp][row] m, then l, then o
    float* part_l = part_m + 4 * kRows;
    float* part_o = part_l + 4 * kRows;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = 16 * t + 8 * half + group_row;
        float sum = l[t][half];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (quad == 0) {
          part_m[warp * kRows + r] = m[t][half];
          part_l[warp * kRows + r] = sum;
        }
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(part_o + (warp * kRows + r) * D + 8 * n + 2 * quad) =
              make_float2(o[t][n][2 * half], o[t][n][2 * half + 1]);
      }
    __syncthreads();
    finish_segment<D, kRows, T>(p, st, cm, [&](int r, int e, float& rm, float& rl, float4& ro) {
      rm = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) rm = fmaxf(rm, part_m[w * kRows + r]);
      const float ref = rm == -INFINITY ? 0.f : rm;
      rl = 0.f;
      ro = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float a = fast_exp2(part_m[w * kRows + r] - ref);
        rl += part_l[w * kRows + r] * a;
        const float4 x = *reinterpret_cast<const float4*>(part_o + (w * kRows + r) * D + e);
        ro.x += x.x * a, ro.y += x.y * a, ro.z += x.z * a, ro.w += x.w * a;
      }
    });
    __syncthreads();
  }
}

// ------------------------------------------------------------ float32, SIMT
//
// float32 products run on the FMA pipes: a thread takes one key of a tile and
// half the block's rows for the scores, then one column and all rows (head_dim
// 128) or half of them (64) for the output.

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
  static constexpr int kOffCommon = kOffO + kRows * D * 4;
  static constexpr int kSmem = kOffCommon + (int)sizeof(Common<kRows>);
};

template <int D>
__global__ void __launch_bounds__(kThreads)
    tree_simt_kernel(const __grid_constant__ TreeParams p) {
  using Sh = SimtShape<D>;
  constexpr int kRows = Sh::kRows, kPitch = Sh::kPitch;
  constexpr int kHalves = kThreads / D;     // threads per output column
  constexpr int kMine = kRows / kHalves;    // rows per thread in the second product
  extern __shared__ __align__(1024) uint8_t smem[];
  auto& cm = *reinterpret_cast<Common<kRows>*>(smem + Sh::kOffCommon);
  float* ks = reinterpret_cast<float*>(smem + Sh::kOffK);
  float* vs = reinterpret_cast<float*>(smem + Sh::kOffV);
  float* qs = reinterpret_cast<float*>(smem + Sh::kOffQ);
  float* ss = reinterpret_cast<float*>(smem + Sh::kOffS);
  float* state_m = reinterpret_cast<float*>(smem + Sh::kOffState);
  float* state_l = state_m + kRows;
  float* state_a = state_l + kRows;
  float* os = reinterpret_cast<float*>(smem + Sh::kOffO);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  griddep_wait();
  griddep_launch_dependents();
  Stretch st = begin_stretch(p, cm);
  while (next_segment(p, cm, st)) {
    const Segment& sg = st.seg;
    prepare_rows<D, kRows, float>(p, sg, cm, warp, lane, [&](int r, int e, const float* x, int n) {
      for (int j = 0; j < n; ++j) qs[r * D + e + j] = x[j];
    });
    if (tid < kRows) state_m[tid] = -INFINITY, state_l[tid] = 0.f;
    float o[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) o[i] = 0.f;
    const float* kbase = static_cast<const float*>(p.key_cache) + sg.b * p.c_sb + sg.h * p.c_sh;
    const float* vbase = static_cast<const float*>(p.value_cache) + sg.b * p.c_sb + sg.h * p.c_sh;
    for (int tile = sg.tile0; tile < sg.tile1; ++tile) {
      const bool tree = tile == sg.tiles - 1;
      if (tree && sg.count == 0) break;
      const int first_key = tree ? sg.length : tile * kTile;
      const int keys = tree ? sg.count : min(kTile, sg.length - first_key);
      __syncthreads();
      if (tree) {
        load_tree_tile<D, float>(p, sg, cm, warp, lane,
                                 [&](int i, int e, const float* k, const float* v, int n) {
                                   for (int j = 0; j < n; ++j) {
                                     ks[i * kPitch + e + j] = k[j];
                                     vs[i * D + e + j] = v[j];
                                   }
                                 });
      } else {
        for (int i = tid; i < kTile * D / 4; i += kThreads) {
          const int row = i / (D / 4), e = i % (D / 4) * 4;
          float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
          if (row < keys) {
            const int64_t at = (int64_t)(first_key + row) * p.c_sp + e;
            k = *reinterpret_cast<const float4*>(kbase + at);
            v = *reinterpret_cast<const float4*>(vbase + at);
          }
          *reinterpret_cast<float4*>(ks + row * kPitch + e) = k;
          *reinterpret_cast<float4*>(vs + row * D + e) = v;
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
          const bool seen = key < keys && (!tree || (cm.mask[r] >> key & 1) != 0);
          const float x = seen ? s[i] * p.scale_log2 : -INFINITY;
          ss[r * kTile + key] = x;
          if (p.weights && key < keys && r < p.rows) score_row(p, sg, r)[first_key + key] = x;
        }
      }
      __syncthreads();
      for (int r = warp; r < kRows; r += kThreads / 32) {
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
      for (int key = 0; key < keys; ++key) {
        const float v = vs[key * D + column];
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const float w = ss[(row0 + i) * kTile + key];
          // An unseen key's value may be infinite or NaN: no product with zero.
          if (!tree || (cm.mask[row0 + i] >> key & 1) != 0) o[i] = fmaf(w, v, o[i]);
        }
      }
    }
    __syncthreads();
    const int column = tid % D, row0 = tid / D * kMine;
#pragma unroll
    for (int i = 0; i < kMine; ++i) os[(row0 + i) * D + column] = o[i];
    __syncthreads();
    finish_segment<D, kRows, float>(p, st, cm,
                                    [&](int r, int e, float& rm, float& rl, float4& ro) {
                                      rm = state_m[r];
                                      rl = state_l[r];
                                      ro = *reinterpret_cast<const float4*>(os + r * D + e);
                                    });
    __syncthreads();
  }
}

// ---------------------------------------------------- the accumulated weights
//
// The attention kernel leaves its scaled scores (base-2) of at most 16 query
// rows per key/value head and each row's log-sum-exp: this one turns a key's
// scores into weights and adds them up, in row order. It moves 4 bytes per row
// and key against the 4 D of the key and value.
constexpr int kWeightThreads = 256;
__global__ void __launch_bounds__(kWeightThreads)
    tree_weights_kernel(const __grid_constant__ TreeParams p) {
  __shared__ float lse[kMaxWeightRows];
  griddep_wait();
  griddep_launch_dependents();
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t unit = (int64_t)b * p.kv_heads + h;
  const RowSpan span = row_span(p, b);
  const int n = span.length + span.count;
  const int j0 = (blockIdx.x * kWeightThreads + threadIdx.x);
  if (threadIdx.x < p.rows) lse[threadIdx.x] = p.lse[unit * p.rows + threadIdx.x];
  __syncthreads();
  if (span.count == 0 || j0 >= n) return;
  float sum = 0.f;
  for (int r = 0; r < p.rows; ++r)
    if (lse[r] != INFINITY)  // an empty row has no weights
      sum += fast_exp2(p.scores[(unit * p.rows + r) * p.score_stride + j0] - lse[r]);
  float* w = p.weights + b * p.w_sb + h * p.w_sh + j0;
  *w = j0 < span.length ? *w + sum : sum;
}

// ------------------------------------------------------------------ host side

template <typename Kernel>
int launch(Kernel kernel, int smem, const TreeParams& p, cudaStream_t stream,
           const char* what) {
  if (int rc = check_cuda(
          cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), what))
    return rc;
  return launch_pdl(kernel, dim3(p.ctas), dim3(kThreads), smem, stream, what, p);
}

// Query rows that one CTA holds against a key tile, by dtype and rows per
// key/value head.
int rows_per_block(int dtype, int rows) {
  if (dtype == ASRBACK_F32) return 16;
  return rows <= 16 ? 16 : 32;
}

struct Plan {
  int block_rows, mblocks, ctas;
  size_t counter_bytes, part_bytes, lse_bytes, score_bytes;
  int64_t score_stride;
  size_t total() const { return counter_bytes + part_bytes + lse_bytes + score_bytes; }
};

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

Plan plan_for(int dtype, int batch, int nodes, int heads, int kv_heads, int head_dim,
              int cache_length, bool weights) {
  Plan plan{};
  const int rows = nodes * (heads / kv_heads);
  plan.block_rows = rows_per_block(dtype, rows);
  plan.mblocks = (rows + plan.block_rows - 1) / plan.block_rows;
  const int64_t items = (int64_t)batch * kv_heads * plan.mblocks;
  const int64_t tiles = items * ((cache_length + kTile - 1) / kTile + 1);
  // Resident CTAs per SM: two of the 16-row kernel (96 KB rings), one of the
  // 32-row kernel's register count.
  const int per_sm = dtype == ASRBACK_BF16 && plan.block_rows == 16 ? 2 : 1;
  plan.ctas = static_cast<int>(std::min<int64_t>(tiles, (int64_t)per_sm * sm_count()));
  plan.counter_bytes = up16(items * sizeof(int));
  plan.part_bytes = up16((size_t)2 * plan.ctas * plan.block_rows * (head_dim + 2) * sizeof(float));
  if (weights) {
    plan.score_stride = (cache_length + 3) / 4 * 4;
    plan.lse_bytes = up16((size_t)batch * kv_heads * rows * sizeof(float));
    plan.score_bytes = (size_t)batch * kv_heads * rows * plan.score_stride * sizeof(float);
  }
  return plan;
}

}  // namespace
}  // namespace asrback

using namespace asrback;
using namespace asrback::tree;

extern "C" size_t asrback_tree_counter_bytes(int dtype, int batch, int nodes, int heads,
                                             int kv_heads) {
  if (batch < 1 || nodes < 1 || kv_heads < 1 || heads < kv_heads) return 0;
  return plan_for(dtype, batch, nodes, heads, kv_heads, 64, 1, false).counter_bytes;
}

extern "C" size_t asrback_tree_workspace_bytes(int dtype, int batch, int nodes, int heads,
                                               int kv_heads, int head_dim, int cache_length,
                                               int with_weights) {
  if (batch < 1 || nodes < 1 || kv_heads < 1 || heads < kv_heads || head_dim < 1 ||
      cache_length < 1)
    return 0;
  const Plan plan = plan_for(dtype, batch, nodes, heads, kv_heads, head_dim, cache_length,
                             with_weights != 0);
  return plan.total() - plan.counter_bytes;
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
    float scale, void* counters, size_t counter_bytes, void* workspace, size_t workspace_bytes,
    int32_t* status, void* stream) {
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
  const int64_t strides[] = {q_stride_batch, q_stride_node, q_stride_head,  k_stride_batch,
                             k_stride_node,  k_stride_head, v_stride_batch, v_stride_node,
                             v_stride_head,  c_stride_batch, c_stride_position, c_stride_head,
                             o_stride_batch, o_stride_node, o_stride_head};
  for (int64_t s : strides)
    if (s < 0 || (s * esize) % 16 != 0)
      return fail(ASRBACK_ERR_ARGUMENT,
                  "strides must not be negative and rows must start on 16-byte boundaries");
  if (rotary && (table_stride * esize) % 16 != 0)
    return fail(ASRBACK_ERR_ARGUMENT, "cos and sin rows must start on 16-byte boundaries");
  const void* pointers[] = {query, key, value, key_cache, value_cache, out, q_norm_weight,
                            k_norm_weight, cos, sin};
  for (const void* ptr : pointers)
    if (!aligned16(ptr)) return fail(ASRBACK_ERR_ARGUMENT, "pointers must be 16-byte aligned");
  if (c_stride_position < head_dim || (kv_heads > 1 && c_stride_head < head_dim) ||
      (heads > 1 && o_stride_head < head_dim) || (nodes > 1 && o_stride_node < head_dim))
    return fail(ASRBACK_ERR_ARGUMENT, "cache or output strides do not hold rows of head_dim");
  const int rows = nodes * (heads / kv_heads);
  if (weights && rows > kMaxWeightRows)
    return fail(ASRBACK_ERR_ARGUMENT,
                "weights take at most %d query rows per key/value head (nodes x heads / kv_heads), "
                "got %d",
                kMaxWeightRows, rows);
  if (weights && kv_heads > 65535)
    return fail(ASRBACK_ERR_ARGUMENT, "weights take at most 65535 key/value heads");
  const Plan plan = plan_for(dtype, batch, nodes, heads, kv_heads, head_dim, cache_length,
                             weights != nullptr);
  if ((int64_t)batch * kv_heads * plan.mblocks * ((cache_length + kTile - 1) / kTile + 1) >
      (int64_t)1 << 30)
    return fail(ASRBACK_ERR_ARGUMENT, "too many key tiles for one call");
  const size_t need = plan.total() - plan.counter_bytes;
  if (!counters || counter_bytes < plan.counter_bytes)
    return fail(ASRBACK_ERR_WORKSPACE, "counters of %zu bytes, %zu needed",
                counters ? counter_bytes : (size_t)0, plan.counter_bytes);
  if (!workspace || workspace_bytes < need)
    return fail(ASRBACK_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed",
                workspace ? workspace_bytes : (size_t)0, need);
  if (!aligned16(workspace) || !aligned16(counters))
    return fail(ASRBACK_ERR_ARGUMENT, "counters and workspace must be 16-byte aligned");

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
  p.rows = rows, p.mblocks = plan.mblocks, p.cache_length = cache_length, p.ctas = plan.ctas;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  p.counters = static_cast<int*>(counters);
  p.parts = reinterpret_cast<float*>(at);
  at += plan.part_bytes;
  p.lse = reinterpret_cast<float*>(at);
  at += plan.lse_bytes;
  p.scores = reinterpret_cast<float*>(at);
  p.score_stride = plan.score_stride;
  p.status = status;

  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc;
  const char* what = "tree attention launch";
  auto mma = [&](auto dim, auto mt, auto held) {
    constexpr int D = decltype(dim)::value, MT = decltype(mt)::value;
    constexpr bool W = decltype(held)::value;
    return launch(tree_mma_kernel<D, MT, W>, MmaShape<D, MT, W>::kSmem, p, s, what);
  };
  using std::integral_constant;
  using one = integral_constant<int, 1>;
  using two = integral_constant<int, 2>;
  auto by_rows = [&](auto dim) {
    if (weights) return mma(dim, one{}, std::true_type{});
    if (plan.block_rows == 16) return mma(dim, one{}, std::false_type{});
    return mma(dim, two{}, std::false_type{});
  };
  if (dtype == ASRBACK_BF16)
    rc = head_dim == 64 ? by_rows(integral_constant<int, 64>{})
                        : by_rows(integral_constant<int, 128>{});
  else if (head_dim == 64)
    rc = launch(tree_simt_kernel<64>, SimtShape<64>::kSmem, p, s, what);
  else
    rc = launch(tree_simt_kernel<128>, SimtShape<128>::kSmem, p, s, what);
  if (rc) return rc;
  if (weights) {
    const dim3 grid((cache_length + kWeightThreads - 1) / kWeightThreads, kv_heads, batch);
    rc = launch_pdl(tree_weights_kernel, grid, dim3(kWeightThreads), 0, s, "tree weights launch", p);
  }
  return rc ? rc : ok();
}
