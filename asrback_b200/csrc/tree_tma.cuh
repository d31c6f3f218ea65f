// TMA side of the bf16 draft-tree attention kernels: tensor maps of the cache and
// the loads of a tile of keys or values.
#pragma once

#include "tcgen05.cuh"
#include "tree_attention.cuh"

namespace asrback {
namespace tree {

constexpr int kTailKeys = 16;  // positions per copy of a row's last tile

// Tensor maps of the cache: ring units (a box of 64 or 128 positions x D) and
// blocks of kTailKeys positions x 64 columns.
struct Maps {
  CUtensorMap tile[2], tail[2];  // keys, values
};

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int c0, int c1, int c2,
                                            int c3, int c4, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4),
      "r"(smem_addr(bar))
      : "memory");
}
// Loads the `keys` positions from `key` on of a row's head as one ring unit of
// kKeys positions, the box of `maps`: a full unit is one copy, of others only the
// blocks of kTailKeys positions that hold keys. One thread calls it.
template <int D, int kKeys = kTile>
__device__ __forceinline__ void load_tile(uint8_t* dst, const Maps& maps, int which, int key,
                                          int keys, int h, int b, uint64_t* bar) {
  if (keys >= kKeys) {
    mbar_arrive_expect_tx(bar, kKeys * D * 2);
    tma_load_5d(dst, &maps.tile[which], 0, key, 0, h, b, bar);
    return;
  }
  const int blocks = (keys + kTailKeys - 1) / kTailKeys;
  mbar_arrive_expect_tx(bar, blocks * kTailKeys * D * 2);
  for (int k = 0; k < blocks * kTailKeys; k += kTailKeys)
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      tc::tma_load_4d(dst + c * kKeys * 128 + k * 128, &maps.tail[which], 64 * c, key + k, h, b,
                      bar);
}

// The cache as a map {64 columns, position, column block, head, row} with a box
// of `unit` positions of all column blocks, and as one {column, position, head, row}
// with a box of 64 columns of kTailKeys positions.
inline int make_maps(CUtensorMap* tile, CUtensorMap* tail, void* base, const TreeParams& p,
                     int head_dim, int unit) {
  int rc = ASRBACK_OK;
  auto encode = tc::tensor_map_encoder(&rc);
  if (!encode) return rc;
  // A dimension of one may have any stride; the encoder wants a plausible one.
  const auto bytes = [&](int64_t stride, int64_t size) {
    return static_cast<cuuint64_t>((size > 1 ? stride : head_dim) * 2);
  };
  const cuuint64_t position = bytes(p.c_sp, p.cache_length), head = bytes(p.c_sh, p.kv_heads),
                   row = bytes(p.c_sb, p.batch);
  const cuuint64_t length = p.cache_length, heads = p.kv_heads, rows = p.batch;
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  const auto make = [&](CUtensorMap* map, int rank, const cuuint64_t* dims,
                        const cuuint64_t* strides, const cuuint32_t* box) {
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, base, dims, strides, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  const cuuint64_t blocks = head_dim / 64;
  const cuuint64_t dims5[5] = {64, length, blocks, heads, rows};
  const cuuint64_t strides5[4] = {position, 128, head, row};
  const cuuint32_t box5[5] = {64, (cuuint32_t)unit, (cuuint32_t)blocks, 1, 1};
  const cuuint64_t dims4[4] = {(cuuint64_t)head_dim, length, heads, rows};
  const cuuint64_t strides4[3] = {position, head, row};
  const cuuint32_t box4[4] = {64, kTailKeys, 1, 1};
  CUresult res = make(tile, 5, dims5, strides5, box5);
  if (res == CUDA_SUCCESS) res = make(tail, 4, dims4, strides4, box4);
  if (res != CUDA_SUCCESS)
    return fail(ASRBACK_ERR_ARGUMENT,
                "cuTensorMapEncodeTiled rejected the cache (error %d): strides (%lld, %lld, %lld)",
                (int)res, (long long)p.c_sb, (long long)p.c_sp, (long long)p.c_sh);
  return ASRBACK_OK;
}

// Both caches' maps, the keys' with units of `key_unit` positions.
inline int make_maps(Maps* maps, const TreeParams& p, int head_dim, int key_unit) {
  if (int rc = make_maps(&maps->tile[0], &maps->tail[0], p.key_cache, p, head_dim, key_unit))
    return rc;
  return make_maps(&maps->tile[1], &maps->tail[1], p.value_cache, p, head_dim, kTile);
}

}  // namespace tree
}  // namespace asrback
