// Attention of a tree of drafted tokens over a key/value cache.
//
// Query of node t of sequence b and query head h attends the first
// kv_lens[b] cache rows of KV head h / G and, of the tree's own keys, those
// of its ancestors and itself (parents[t] < t; a node whose parent is not
// one has only itself):
//   o = sum_n p_n v_n,  p = softmax(scale * q . k_n) over those keys,
// with the base-2 log-sum-exp (scale included) as the optional statistic.
// Nodes past a sequence's tree_sizes[b] give o = 0 and lse = -inf.
//
// One warp per query row, lanes across the head, keys in order: online
// softmax in base 2.
#include "attn_launch.h"
#include "sm100_primitives.cuh"

namespace tk {
namespace {

constexpr int kMaxWords = kTreeMaxNodes / 32;

template <bool kBf16>
__device__ __forceinline__ float from16(uint16_t h) {
  if constexpr (kBf16) {
    return __uint_as_float(static_cast<uint32_t>(h) << 16);
  } else {
    return __half2float(__ushort_as_half(h));
  }
}

template <bool kBf16>
__global__ void __launch_bounds__(256) tree_attn_kernel(const TreeAttnArgs a) {
  const int lane = threadIdx.x & 31;
  const long long row = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (row >= a.B * a.Hkv * a.G * a.T) return;
  const int t = static_cast<int>(row % a.T);
  const long long head = row / a.T;
  const long long b = head / (a.Hkv * a.G);
  const int h = static_cast<int>(head % (a.Hkv * a.G) / a.G);
  const int D = static_cast<int>(a.D);
  const int len = min(max(a.kv_lens[b], 0), static_cast<int>(a.L));
  const int size = a.tree_sizes != nullptr ? min(max(a.tree_sizes[b], 0), static_cast<int>(a.T)) : static_cast<int>(a.T);
  uint16_t* o = static_cast<uint16_t*>(a.o) + row * D;
  float qr[4], acc[4];
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + row * D;
  for (int i = 0; i < 4; ++i) {
    const int c = lane + 32 * i;
    qr[i] = c < D ? from16<kBf16>(q[c]) * a.scale_log2 : 0.0f;
    acc[i] = 0.0f;
  }
  uint32_t seen[kMaxWords] = {};
  if (t < size) {
    int node = t;
    while (node >= 0) {
      seen[node >> 5] |= 1u << (node & 31);
      const int up = a.parents != nullptr ? a.parents[b * a.parent_stride + node] : node - 1;
      node = up < node ? up : -1;
    }
  }
  float m = -INFINITY, l = 0.0f;
  for (int n = 0; t < size && n < len + t + 1; ++n) {
    const bool on_cache = n < len;
    const int j = n - len;
    if (!on_cache && !((seen[j >> 5] >> (j & 31)) & 1u)) continue;
    const int64_t* ks = a.strides + (on_cache ? 0 : 6);
    const int64_t* vs = ks + 3;
    const int64_t r = on_cache ? n : j;
    const uint16_t* k = static_cast<const uint16_t*>(on_cache ? a.k : a.k_tree) + b * ks[0] + h * ks[1] + r * ks[2];
    const uint16_t* v = static_cast<const uint16_t*>(on_cache ? a.v : a.v_tree) + b * vs[0] + h * vs[1] + r * vs[2];
    float x = 0.0f;
    for (int i = 0; i < 4; ++i) {
      const int c = lane + 32 * i;
      if (c < D) x += qr[i] * from16<kBf16>(k[c]);
    }
    for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
    const float m_new = fmaxf(m, x);
    const float alpha = ex2(m - m_new), p = ex2(x - m_new);
    m = m_new;
    l = l * alpha + p;
    for (int i = 0; i < 4; ++i) {
      const int c = lane + 32 * i;
      if (c < D) acc[i] = acc[i] * alpha + p * from16<kBf16>(v[c]);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  for (int i = 0; i < 4; ++i) {
    const int c = lane + 32 * i;
    if (c < D) o[c] = static_cast<uint16_t>(pack2<kBf16>(acc[i] * inv, 0.0f) & 0xffffu);
  }
  if (a.lse != nullptr && lane == 0) a.lse[row] = t < size ? m + lg2(l) : -INFINITY;
}

}  // namespace

int launch_tree_attn(const TreeAttnArgs& a) {
  const long long rows = a.B * a.Hkv * a.G * a.T;
  const unsigned grid = static_cast<unsigned>((rows + 7) / 8);
  if (a.bf16)
    tree_attn_kernel<true><<<grid, 256, 0, a.stream>>>(a);
  else
    tree_attn_kernel<false><<<grid, 256, 0, a.stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

}  // namespace tk
