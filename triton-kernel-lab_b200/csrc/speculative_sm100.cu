// Speculative decoding around the attention: acceptance of drafted tokens
// against the target's probabilities, and the write of the accepted tokens'
// keys and values into the cache.
//
// Verification.  Node 0 is the sequence's last known token; node c > 0
// carries a drafted token x_c that continues its parent n (parents[c] < c; a
// chain has n = c - 1).  p_n is the target's distribution after node n.  From
// node 0, the children of the current node are tried in index order with the
// given uniform numbers u_c in [0, 1):
//   exact drafts (no draft probabilities): accepted if u_c (1 - S_c) < p_n(x_c),
//     S_c the mass under p_n of the earlier siblings' (different) tokens; a
//     token tried before has nothing left and is refused;
//   drafts drawn from q_n (chains only): accepted if u_c q_n(x_c) < p_n(x_c).
// The walk goes on from an accepted child.  At the last accepted node n the
// next token is the winner of an exponential race, argmax_v w_v / e_v, with
// the residual weights w = p_n without the tried tokens, max(p_n - q_n, 0),
// or p_n where n has no child; p_n also where the residual has no mass left.
// The emitted tokens are then distributed as the target's own samples.
//
// Whether child c passes depends on its siblings alone, so every node is
// tested at once and the walk only follows the chosen children.
#include "attn_launch.h"
#include "sm100_primitives.cuh"

namespace tk {
namespace {

template <int kType>
__device__ __forceinline__ float prob_at(const void* p, int64_t i) {
  if constexpr (kType == kProbF32) {
    return static_cast<const float*>(p)[i];
  } else if constexpr (kType == kProbBf16) {
    return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
  } else {
    return __half2float(static_cast<const __half*>(p)[i]);
  }
}

__device__ __forceinline__ long long token_at(const VerifyArgs& a, int64_t i) {
  return a.tokens_64 ? static_cast<const long long*>(a.tokens)[i] : static_cast<const int*>(a.tokens)[i];
}

constexpr int kVerifyThreads = 1024;

// One CTA per sequence.
template <int kType>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyArgs a) {
  __shared__ int s_parent[kTreeMaxNodes], s_child[kTreeMaxNodes];
  __shared__ long long s_token[kTreeMaxNodes];
  __shared__ float s_prob[kTreeMaxNodes];
  __shared__ unsigned char s_pass[kTreeMaxNodes];
  __shared__ int s_last;
  __shared__ float s_score[32];
  __shared__ int s_index[32];
  const int64_t b = blockIdx.x;
  const int T = static_cast<int>(a.T), V = static_cast<int>(a.V);
  const int size = a.tree_sizes != nullptr ? min(max(a.tree_sizes[b], 0), T) : T;
  for (int c = threadIdx.x; c < T; c += blockDim.x) {
    int n = c - 1;
    if (a.parents != nullptr && c > 0) n = a.parents[b * a.parent_stride + c];
    if (n >= c || n < 0 || c >= size) n = -1;  // hangs on nothing: never reached
    const long long x = token_at(a, b * T + c);
    const bool real = n >= 0 && x >= 0 && x < V;
    s_parent[c] = n;
    s_token[c] = x;
    s_prob[c] = real ? prob_at<kType>(a.target, b * a.target_stride[0] + n * a.target_stride[1] + x) : 0.0f;
    s_child[c] = -1;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < T; c += blockDim.x) {
    bool pass = false;
    const int n = s_parent[c];
    if (n >= 0 && s_prob[c] > 0.0f) {
      const float u = a.uniforms[b * T + c];
      if (a.draft != nullptr) {
        const float q = prob_at<kType>(a.draft, b * a.draft_stride[0] + n * a.draft_stride[1] + s_token[c]);
        pass = u * q < s_prob[c];
      } else {
        float mass = 0.0f;
        bool again = false;
        for (int s = n + 1; s < c; ++s) {
          if (s_parent[s] != n) continue;
          if (s_token[s] == s_token[c]) again = true;
          bool first = true;
          for (int r = n + 1; r < s; ++r) first = first && !(s_parent[r] == n && s_token[r] == s_token[s]);
          if (first) mass += s_prob[s];
        }
        pass = !again && u * fmaxf(1.0f - mass, 0.0f) < s_prob[c];
      }
    }
    s_pass[c] = pass;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < T; c += blockDim.x) {
    if (!s_pass[c]) continue;
    const int n = s_parent[c];
    bool first = true;
    for (int s = n + 1; s < c; ++s) first = first && !(s_parent[s] == n && s_pass[s]);
    if (first) s_child[n] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int last = -1, length = 0;
    for (int n = size > 0 ? 0 : -1; n >= 0; n = s_child[n]) {
      a.path[b * T + length++] = n;
      last = n;
    }
    a.path_lens[b] = length;
    for (int i = length; i < T; ++i) a.path[b * T + i] = -1;
    s_last = last;
  }
  __syncthreads();
  const int last = s_last;
  if (last < 0) {
    if (threadIdx.x == 0) {
      if (a.tokens_64)
        static_cast<long long*>(a.next)[b] = -1;
      else
        static_cast<int*>(a.next)[b] = -1;
    }
    return;
  }
  bool has_child = false;
  for (int c = last + 1; c < size; ++c) has_child = has_child || s_parent[c] == last;
  const int64_t row = b * a.target_stride[0] + last * a.target_stride[1];
  const int64_t drow = a.draft != nullptr ? b * a.draft_stride[0] + last * a.draft_stride[1] : 0;
  for (int attempt = 0; attempt < 2; ++attempt) {
    const bool residual = attempt == 0 && has_child;
    float best = 0.0f;
    int index = INT_MAX;
    for (int v = threadIdx.x; v < V; v += blockDim.x) {
      float w = prob_at<kType>(a.target, row + v);
      if (residual) {
        if (a.draft != nullptr) {
          w -= prob_at<kType>(a.draft, drow + v);
        } else {
          for (int c = last + 1; c < size; ++c)
            if (s_parent[c] == last && s_token[c] == v) w = 0.0f;
        }
      }
      if (!(w > 0.0f)) continue;
      const float score = __fdiv_rn(w, a.noise[b * V + v]);
      if (score > best) {
        best = score;
        index = v;
      }
    }
    for (int off = 16; off > 0; off >>= 1) {
      const float s = __shfl_xor_sync(0xffffffffu, best, off);
      const int i = __shfl_xor_sync(0xffffffffu, index, off);
      if (s > best || (s == best && i < index)) {
        best = s;
        index = i;
      }
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      s_score[threadIdx.x >> 5] = best;
      s_index[threadIdx.x >> 5] = index;
    }
    __syncthreads();
    best = 0.0f;
    index = INT_MAX;
    for (int i = 0; i < kVerifyThreads / 32; ++i)
      if (s_score[i] > best || (s_score[i] == best && s_index[i] < index)) {
        best = s_score[i];
        index = s_index[i];
      }
    if (index != INT_MAX || !residual) {
      if (threadIdx.x == 0) {
        const int next = index != INT_MAX ? index : 0;
        if (a.tokens_64)
          static_cast<long long*>(a.next)[b] = next;
        else
          static_cast<int*>(a.next)[b] = next;
      }
      return;
    }
  }
}

// One CTA per (sequence and layer, head): the accepted rows, 16 bytes a thread.
__global__ void __launch_bounds__(128) commit_kernel(const CommitArgs a) {
  const int64_t b = blockIdx.x % a.B, layer = blockIdx.x / a.B, h = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const int n = min(max(a.path_lens[b], 0), static_cast<int>(a.T));
  const int start = min(max(a.kv_lens[b], 0), static_cast<int>(a.L));
  const int fit = min(n, static_cast<int>(a.L) - start);
  if (blockIdx.y == 0 && layer == 0 && !is_v && threadIdx.x == 0) {
    a.new_lens[b] = start + fit;
    if (fit < n) atomicCAS(a.status, kOk, kErrTooLarge);
  }
  const int64_t* cs = a.strides + (is_v ? 4 : 0);
  const int64_t* ts = a.strides + (is_v ? 12 : 8);
  uint16_t* dst = static_cast<uint16_t*>(is_v ? a.v : a.k) + layer * cs[0] + b * cs[1] + h * cs[2];
  const uint16_t* src = static_cast<const uint16_t*>(is_v ? a.v_tree : a.k_tree) + layer * ts[0] + b * ts[1] + h * ts[2];
  const int chunks = static_cast<int>(a.D / 8);
  for (int u = threadIdx.x; u < fit * chunks; u += blockDim.x) {
    const int i = u / chunks, c = u % chunks * 8;
    const int node = a.path[b * a.T + i];
    if (node < 0 || node >= a.T) {
      atomicCAS(a.status, kOk, kErrInvalidArgument);
      continue;
    }
    *reinterpret_cast<uint4*>(dst + (start + i) * cs[3] + c) = *reinterpret_cast<const uint4*>(src + node * ts[3] + c);
  }
}

}  // namespace

int launch_verify(const VerifyArgs& a) {
  const unsigned grid = static_cast<unsigned>(a.B);
  if (a.type == kProbF32)
    verify_kernel<kProbF32><<<grid, kVerifyThreads, 0, a.stream>>>(a);
  else if (a.type == kProbBf16)
    verify_kernel<kProbBf16><<<grid, kVerifyThreads, 0, a.stream>>>(a);
  else
    verify_kernel<kProbF16><<<grid, kVerifyThreads, 0, a.stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

int launch_commit(const CommitArgs& a) {
  const dim3 grid(static_cast<unsigned>(a.layers * a.B), static_cast<unsigned>(a.H), 2);
  commit_kernel<<<grid, 128, 0, a.stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

}  // namespace tk
