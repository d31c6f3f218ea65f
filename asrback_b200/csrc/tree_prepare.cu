// What comes before the draft-tree attention's products, sm_100a: the query rows
// normalised, rotated and laid out as the products read them, and the nodes'
// keys and values, normalised and rotated likewise, written to the cache.
//
// One pass over the call's inputs, a few MB at most, so latency bounds it: every
// row is a group of D / 16 lanes, all rows run at once, and the attention kernel
// is launched with it (programmatic dependent launch) and streams the cached
// keys meanwhile, which this one does not touch. Measured: 64 rows x 16 nodes, 32
// heads of 128 in all (17 MB) 3 us behind the kernel before it, 8 rows x 64 nodes
// 5 us.
#include "capi_internal.h"
#include "tree_attention.cuh"

namespace asrback {
namespace {

using namespace tree;

constexpr int kThreads = 128;

// Rows being prepared are shared out over D / 16 lanes each: lane c of a row
// holds elements 8c .. 8c+7 and their rotary partners D/2 + 8c .. + 7, so that
// the rotation needs no other lane and the norm three shuffles at most.
template <typename T>
struct Octet;  // eight elements as loaded
template <>
struct Octet<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const void* row, int element) {
    u = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(row) + element));
  }
  __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void copy(void* row, int element) const {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(row) + element) = u;
  }
  __device__ __forceinline__ float operator[](int i) const {
    const uint32_t w = i < 2 ? u.x : i < 4 ? u.y : i < 6 ? u.z : u.w;
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
  __device__ __forceinline__ static void store(void* row, int element, const float* x) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(row) + element) =
        *reinterpret_cast<uint4*>(h);
  }
};
template <>
struct Octet<float> {
  float4 u[2];
  __device__ __forceinline__ void load(const void* row, int element) {
    const float4* at = reinterpret_cast<const float4*>(static_cast<const float*>(row) + element);
    u[0] = __ldg(at), u[1] = __ldg(at + 1);
  }
  __device__ __forceinline__ void zero() { u[0] = u[1] = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void copy(void* row, int element) const {
    float4* at = reinterpret_cast<float4*>(static_cast<float*>(row) + element);
    at[0] = u[0], at[1] = u[1];
  }
  __device__ __forceinline__ float operator[](int i) const {
    const float4 q = u[i >> 2];
    return (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
  }
  __device__ __forceinline__ static void store(void* row, int element, const float* x) {
    float4* at = reinterpret_cast<float4*>(static_cast<float*>(row) + element);
    at[0] = make_float4(x[0], x[1], x[2], x[3]);
    at[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
};

template <int D, typename T>
struct RowSlice {
  static constexpr int kLanes = D / 16;  // lanes per row
  Octet<T> half[2];
  __device__ __forceinline__ void load(const void* row, int c) {
    half[0].load(row, 8 * c);
    half[1].load(row, D / 2 + 8 * c);
  }
  __device__ __forceinline__ void zero() { half[0].zero(), half[1].zero(); }
  __device__ __forceinline__ void unpack(float* x) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = half[i >> 3][i & 7];
  }
};

// RMSNorm, then rotate-half rotary embedding of a row, all in float32.
template <int D, typename T>
__device__ __forceinline__ void norm_rotate(float eps, const RowSlice<D, T>& w,
                                            const RowSlice<D, T>& cs, const RowSlice<D, T>& sn,
                                            float* x) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
  for (int o = RowSlice<D, T>::kLanes / 2; o > 0; o >>= 1)
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float r = rsqrtf(ss / D + eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x[i] * r * w.half[0][i], b = x[i + 8] * r * w.half[1][i];
    x[i] = a * cs.half[0][i] - b * sn.half[0][i];
    x[i + 8] = b * cs.half[1][i] + a * sn.half[1][i];
  }
}

// Row tasks of a batch row: the query rows of its blocks (rows past the last
// query row included, as zeros), then a key and value row per (head, node).
// kSplit: q is multiplied by the softmax scale (base 2) and taken apart into two
// bf16 parts, so that rounding it costs the scores 2^-17 and not 2^-9.
template <int D, typename T, bool kSplit>
__global__ void __launch_bounds__(kThreads)
    tree_prepare_kernel(const __grid_constant__ TreeParams p) {
  using Slice = RowSlice<D, T>;
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.y, c = threadIdx.x % Slice::kLanes;
  const int task = blockIdx.x * (kThreads / Slice::kLanes) + threadIdx.x / Slice::kLanes;
  const int block_rows = p.block_rows;
  const int q_rows = p.kv_heads * p.mblocks * block_rows;
  const bool query = task < q_rows;
  // A query row's block, row of the block and node; or a key's head and node.
  int block = 0, r = 0, h = 0, node = 0, head = 0;
  bool in = false;
  if (query) {
    block = task / block_rows;
    r = task % block_rows;
    h = block / p.mblocks;
    const int row = block % p.mblocks * block_rows + r;
    node = row / p.group;
    head = h * p.group + row % p.group;
    in = row < p.rows;
  } else {
    h = (task - q_rows) / p.nodes;
    node = (task - q_rows) % p.nodes;
    in = h < p.kv_heads;
  }
  // All loads that need nothing else go out together, whether or not the node
  // turns out to be live; the angles follow the positions.
  unsigned long long mask = 0;
  int depth = 0;
  Slice x_in, v_in, w, cs, sn;
  x_in.zero(), v_in.zero(), w.zero(), cs.zero(), sn.zero();
  if (in) {
    const int64_t at = (int64_t)b * p.nodes + node;
    mask = static_cast<unsigned long long>(__ldg(p.ancestors + at));
    if (query) {
      x_in.load(static_cast<const T*>(p.q) + b * p.q_sb + node * p.q_sn + head * p.q_sh, c);
    } else {
      x_in.load(static_cast<const T*>(p.k) + b * p.k_sb + node * p.k_sn + h * p.k_sh, c);
      v_in.load(static_cast<const T*>(p.v) + b * p.v_sb + node * p.v_sn + h * p.v_sh, c);
    }
    if (p.q_norm) {
      w.load(query ? p.q_norm : p.k_norm, c);
      // A valid plan's depth is at most the node's index; any other stays in
      // the table.
      depth = min(max(__ldg(p.depths + at), 0), node);
    }
  }
  const RowSpan span = row_span(p, b);
  if (span.bad && blockIdx.x == 0 && threadIdx.x == 0 && p.status)
    atomicOr(p.status, ASRBACK_STATUS_POSITION);
  in = in && node < span.count;
  mask = in ? mask & (span.count >= 64 ? ~0ull : (1ull << span.count) - 1) : 0;
  if (in && p.q_norm) {
    const int64_t place = __ldg(p.positions + b) + depth;
    cs.load(static_cast<const T*>(p.cos) + place * p.table_stride, c);
    sn.load(static_cast<const T*>(p.sin) + place * p.table_stride, c);
  }
  float x[16];
  x_in.unpack(x);
  if (p.q_norm) norm_rotate<D, T>(p.eps, w, cs, sn, x);
  if (!query) {
    if (!in) return;
    // A node without a bit writes nothing; what lies in its slot may be anything.
    bool odd = mask == 0;
    if (mask != 0) {
      const int64_t to = b * p.c_sb + (int64_t)(span.length + node) * p.c_sp + h * p.c_sh;
      T* key = static_cast<T*>(p.key_cache) + to;
      T* value = static_cast<T*>(p.value_cache) + to;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        Octet<T>::store(key, half * (D / 2) + 8 * c, x + 8 * half);
        v_in.half[half].copy(value, half * (D / 2) + 8 * c);
#pragma unroll
        for (int i = 0; i < 8; ++i) odd |= !(fabsf(v_in.half[half][i]) < INFINITY);
      }
    }
    // Whether any lane of the row (lanes leave together) found one.
    const unsigned mine = ((1u << (Slice::kLanes - 1)) * 2u - 1u)
                          << ((threadIdx.x & 31) / Slice::kLanes * Slice::kLanes);
    odd = __any_sync(mine, odd);
    // The flag goes to each of the head's blocks.
    for (int i = c; i < p.mblocks; i += Slice::kLanes) {
      uint8_t* next = p.q_blocks + (((int64_t)b * p.kv_heads + h) * p.mblocks + i + 1) *
                                       p.q_block_bytes;
      (next - kMaxNodes)[node] = odd;
    }
    return;
  }
  if (mask == 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;
  }
  uint8_t* out = p.q_blocks + ((int64_t)b * p.kv_heads * p.mblocks + block) * p.q_block_bytes;
  if (c == 0)
    reinterpret_cast<unsigned long long*>(out + p.q_block_bytes - kMaxNodes)[r - block_rows] = mask;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int e = half * (D / 2) + 8 * c;
    if constexpr (sizeof(T) == 4) {
      Octet<T>::store(reinterpret_cast<T*>(out) + r * D, e, x + 8 * half);
    } else {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a0 = x[8 * half + 2 * j], a1 = x[8 * half + 2 * j + 1];
        if constexpr (kSplit) a0 *= p.scale_log2, a1 *= p.scale_log2;
        const __nv_bfloat162 top = __floats2bfloat162_rn(a0, a1);
        hi[j] = *reinterpret_cast<const uint32_t*>(&top);
        const __nv_bfloat162 rest = __floats2bfloat162_rn(a0 - __uint_as_float(hi[j] << 16),
                                                          a1 - __uint_as_float(hi[j] & 0xffff0000u));
        lo[j] = *reinterpret_cast<const uint32_t*>(&rest);
      }
      uint8_t* to = out + tile_at(block_rows, r, e / 8);
      *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if constexpr (kSplit)
        *reinterpret_cast<uint4*>(to + block_rows * D * 2) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  }
}

template <int D, typename T, bool kSplit>
int launch(const TreeParams& p, cudaStream_t stream) {
  constexpr int kPerCta = kThreads / RowSlice<D, T>::kLanes;
  const int tasks = p.kv_heads * (p.mblocks * p.block_rows + p.nodes);
  return launch_pdl(tree_prepare_kernel<D, T, kSplit>,
                    dim3((tasks + kPerCta - 1) / kPerCta, p.batch), dim3(kThreads), 0, stream,
                    "tree preparation launch", p);
}

}  // namespace

namespace tree {

int launch_prepare(int dtype, int head_dim, const TreeParams& p, cudaStream_t stream) {
  using bf16 = __nv_bfloat16;
  if (dtype == ASRBACK_F32)
    return head_dim == 64 ? launch<64, float, false>(p, stream)
                          : launch<128, float, false>(p, stream);
  if (p.q_norm)
    return head_dim == 64 ? launch<64, bf16, true>(p, stream)
                          : launch<128, bf16, true>(p, stream);
  return head_dim == 64 ? launch<64, bf16, false>(p, stream)
                        : launch<128, bf16, false>(p, stream);
}

}  // namespace tree
}  // namespace asrback
